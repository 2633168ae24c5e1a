// Attention over visible key ranges for sm_100a (tcgen05 + TMEM + TMA), backward.
//
//   P  = 2^(a log2 e - lse2),  dP = dO V^T,  dS = P (dP - delta) (1 - (u / cap)^2),  delta_i = dO_i . o_i
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels that each own their outputs, so no gradient is summed with atomics and the results do
// not depend on the order in which CTAs run; each recomputes S and dP (seven tile products where one
// kernel with an atomic dQ has five):
//   dQ:     one CTA per (128 queries, query head, batch), over key steps of 64
//   dK, dV: one CTA per (128 keys, key head, batch), over the query heads of the group and query tiles
// Both keep their accumulators in TMEM and feed dS (and P^T) to the tensor cores from TMEM, written by
// the softmax warps over the scores they were computed from.
//
// delta is formed in the dQ kernel, from the rounded o, and is off by what that rounding does.  The
// row's sum of P (dP - delta) would be zero with the true one: the dQ kernel adds it up as it goes,
// and the dK / dV kernel behind it gets the corrected delta.
#include "doc_attn.cuh"

namespace oxi {
namespace {

// ------------------------------------------------------------------ dQ
constexpr int DQ_KEYS = 64;
constexpr int DQ_THREADS = 320;  // TMA warp, MMA warp, 8 softmax warps: 32 query rows x 32 keys each

template <int DQP, int DVP>
struct DaDqSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int QBLK = DA_TILE * 128, KBLK = DQ_KEYS * 128;
  static constexpr int Q_BYTES = KBQ * QBLK, DO_BYTES = KBV * QBLK, K_BYTES = KBQ * KBLK, V_BYTES = KBV * KBLK;
  static constexpr int KST = 2, VST = 1;  // K_i is held until its dQ product, V_i only until dP_i
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_DO = OFF_Q + Q_BYTES;
  static constexpr int OFF_K = OFF_DO + DO_BYTES;
  static constexpr int OFF_V = OFF_K + KST * K_BYTES;
  static constexpr int OFF_BAR = OFF_V + VST * V_BYTES;
  // two CTAs of the widest heads fill the SM's shared memory: there is no room to align the base by
  // hand, it has to be on a 1024-byte boundary (the kernel checks)
  static constexpr int TOTAL = OFF_BAR + 256;
  static_assert(2 * (TOTAL + 1024) <= 233472, "two CTAs per SM");
};

// Two CTAs on an SM: one's softmax runs while the tensor cores work for the other.  TMEM: dQ, S, dP (then
// dS): S is free for the next step as soon as it has been read, so that the next S is formed while this
// step's exponentials are.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DQ_THREADS, 2)
    da_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, DaParams p,
                 DaTensor o_in, DaTensor do_in, const float* __restrict__ lse2, float* __restrict__ delta,
                 __nv_bfloat16* __restrict__ dq, int64_t ld) {
  using L = DaDqSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) record_error(p.status, OXI_ERR_BOUNDS);
    return;
  }
  uint8_t *sQ = smem + L::OFF_Q, *sDO = smem + L::OFF_DO, *sK = smem + L::OFF_K, *sV = smem + L::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;   // [2]
  uint64_t* k_empty = bars + 3;  // [2]
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 6;
  uint64_t* s_full = bars + 7;
  uint64_t* dp_full = bars + 8;
  uint64_t* ds_full = bars + 9;
  uint64_t* all_done = bars + 10;
  uint64_t* s_free = bars + 11;  // S has been read into registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int qt = gridDim.z - 1 - blockIdx.z, h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (p.Hq / p.Hk);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(s_free, 8);
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  const TileRange kr = key_steps(p, b, qt, DQ_KEYS);
  const int n = kr.end - kr.begin;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t TM_DQ = tmem, TM_S = tmem + 128, TM_DP = tmem + 192;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_full, L::Q_BYTES + L::DO_BYTES);
#pragma unroll
      for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sQ + kb * L::QBLK, &tmQ, q_full, kb * 64, h, qt * DA_TILE, b);
#pragma unroll
      for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sDO + kb * L::QBLK, &tmDO, q_full, kb * 64, h, qt * DA_TILE, b);
      int ki = 0, vi = 0;
      for (; ki < n; ++ki) {
        const int st = ki % L::KST;
        if (!mbar_wait(&k_empty[st], ((ki / L::KST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(&k_full[st], L::K_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sK + st * L::K_BYTES + kb * L::KBLK, &tmK, &k_full[st], kb * 64, hk, (kr.begin + ki) * DQ_KEYS, b);
        // V_{j} behind K_{j+1}
        bool ok = true;
        for (; ok && vi < n && (vi < ki || ki == n - 1); ++vi) {
          ok = mbar_wait(v_empty, (vi & 1) ^ 1, abort_flag, p.status);
          if (!ok) break;
          mbar_arrive_expect_tx(v_full, L::V_BYTES);
#pragma unroll
          for (int kb = 0; kb < L::KBV; ++kb)
            tma_load_4d(sV + kb * L::KBLK, &tmV, v_full, kb * 64, hk, (kr.begin + vi) * DQ_KEYS, b);
        }
        if (!ok) { ++ki; break; }
      }
      mbar_wait(q_full, 0, nullptr, p.status);
      for (int i = max(0, ki - L::KST); i < ki; ++i) mbar_wait(&k_full[i % L::KST], (i / L::KST) & 1, nullptr, p.status);
      if (vi > 0) mbar_wait(v_full, (vi - 1) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t lead = elect_lead();
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, DQ_KEYS, false, false);
      constexpr uint32_t ID_Q = umma_idesc_bf16(DA_TILE, DQP, false, true);
      const int nkq = (p.Dqk + 15) / 16, nkv = (p.Dv + 15) / 16;
      const DaDesc dQ = da_desc(smem_u32(sQ), 16), dDO = da_desc(smem_u32(sDO), 16), dV = da_desc(smem_u32(sV), 16);
      bool ok = warp_wait(q_full, 0, abort_flag, p.status);
      auto issue_s = [&](int i) -> bool {
        if (!warp_wait(&k_full[i % L::KST], (i / L::KST) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        da_mma_kk<DQP, L::QBLK, L::KBLK>(lead, TM_S, dQ, da_desc(smem_u32(sK + (i % L::KST) * L::K_BYTES), 16), ID_S, nkq);
        da_commit(lead, s_full);
        return true;
      };
      // over dS_{i-1}, read by the product issued just before
      auto issue_dp = [&](int i) -> bool {
        if (!warp_wait(v_full, i & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        da_mma_kk<DVP, L::QBLK, L::KBLK>(lead, TM_DP, dDO, dV, ID_S, nkv);
        da_commit(lead, dp_full);
        da_commit(lead, v_empty);
        return true;
      };
      if (ok) ok = issue_s(0) && issue_dp(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && (!warp_wait(s_free, i & 1, abort_flag, p.status) || !issue_s(i + 1))) { ok = false; break; }
        if (!warp_wait(ds_full, i & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const DaDesc dK = da_desc(smem_u32(sK + (i % L::KST) * L::K_BYTES), L::KBLK);
#pragma unroll
        for (int kk = 0; kk < DQ_KEYS / 16; ++kk)  // keys 0..31 in columns 0..15, 32..63 in columns 32..47
          da_mma_ts(lead, TM_DQ, TM_DP + (kk >> 1) * 32 + (kk & 1) * 8, dK.at(kk * 2048), ID_Q,
                    (i | kk) != 0);
        da_commit(lead, &k_empty[i % L::KST]);
        if (i + 1 < n) ok = issue_dp(i + 1);
        else da_commit(lead, all_done);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int r = quarter * 32 + lane;
    const int qpos = qt * DA_TILE + r;
    const TileRange vis = key_range(p, b, qpos);
    const int all_lo = __reduce_max_sync(0xffffffffu, vis.begin), all_hi = __reduce_min_sync(0xffffffffu, vis.end);
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = TM_S + lane_base + half * 32, dp_addr = TM_DP + lane_base + half * 32;
    const bool in = qpos < p.S;
    const int64_t vi = ((int64_t)b * p.Hq + h) * p.S + qpos;
    const float ls = in ? lse2[vi] : INFINITY;
    float dl = 0.f;  // delta of the row, formed while the first tiles load
    if (in) {
      const __nv_bfloat16* orow = reinterpret_cast<const __nv_bfloat16*>(o_in.ptr) + b * o_in.sb + qpos * o_in.ss + h * o_in.sh;
      const __nv_bfloat16* drow = reinterpret_cast<const __nv_bfloat16*>(do_in.ptr) + b * do_in.sb + qpos * do_in.ss + h * do_in.sh;
      for (int c = 0; c < p.Dv; c += 8) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(orow + c)), y = __ldg(reinterpret_cast<const uint4*>(drow + c));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack_bf16(xw[e]), g = unpack_bf16(yw[e]);
          dl = fmaf(a.x, g.x, fmaf(a.y, g.y, dl));
        }
      }
    }
    const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
    const float C = ALIBI ? 1.f : p.c_log2;
    float rest = 0.f;  // sum of P (dP - delta) over this thread's keys
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int k0 = (kr.begin + i) * DQ_KEYS + half * 32;
      const bool padded = tile_has_pad(p, b, k0 / DA_TILE);
      if (!mbar_wait(s_full, i & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[32];
      tmem_ld32(s_addr, x);
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      const bool masked = !(all_lo <= k0 && k0 + 32 <= all_hi);
      const uint32_t bits = masked ? range_bits(vis.begin, vis.end, k0) : 0xffffffffu;
      const float fd = (float)(qpos - k0);
      float f[CAP ? 32 : 1];
      if (CAP) {
        if (warp_near<32>(x, p.x_scale)) {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(tanh_near(__uint_as_float(x[e]) * p.x_scale, f[e]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(tanh_wide(__uint_as_float(x[e]) * p.x_scale, f[e]));
        }
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        float v = __uint_as_float(x[e]);
        if (ALIBI) v = fmaf(-slope2, fabsf(fd - (float)e), v * p.c_log2);
        x[e] = __float_as_uint(ex2_approx(fmaf(v, C, -ls)));
      }
      if (!mbar_wait(dp_full, i & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t d[16], pk[8];
        tmem_ld16(dp_addr + c * 16, d);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int t = c * 16 + e;
          float g = __uint_as_float(x[t]) * (__uint_as_float(d[e]) - dl);
          if (masked) g = ((bits >> t) & 1u) ? g : 0.f;
          rs[e & 1] += g;
          if (CAP) {
            g *= f[t];
            if (masked) g = ((bits >> t) & 1u) ? g : 0.f;  // a hidden score may be NaN, and f with it
          }
          d[e] = __float_as_uint(g);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) pk[e] = pack_bf16(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1]));
        tmem_st8(dp_addr + c * 8, pk);
      }
      rest += rs[0] + rs[1];
      // S_i has read K_i: rows of padding become zero before the dQ product reads them
      if (padded)
        zero_pad_rows<L::KBQ, DQ_KEYS>(sK + (i % L::KST) * L::K_BYTES, p, b, (kr.begin + i) * DQ_KEYS, half * 128 + r, 256);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && n > 0 && !mbar_wait(all_done, 0, abort_flag, p.status)) ok = false;
    // the halves' rests meet in shared memory: every product has completed, so K's ring is free
    float* s_rest = reinterpret_cast<float*>(sK);
    if (ok) s_rest[half * DA_TILE + r] = rest;
    asm volatile("bar.sync 1, 256;" ::: "memory");  // reached by every softmax warp
    if (ok) {
      tc_fence_after();
      if (half == 0 && in) delta[vi] = dl + (s_rest[r] + s_rest[DA_TILE + r]);
      __nv_bfloat16* row = dq + ((int64_t)b * p.S + qpos) * ld + (int64_t)h * p.Dqk;
#pragma unroll 1
      for (int c = half; c < DQP / 32; c += 2) {
        uint32_t w[32];
        if (n > 0) {
          tmem_ld32(TM_DQ + lane_base + c * 32, w);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) w[e] = 0u;
        }
        if (in) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (c * 32 + q * 8 < p.Dqk) {
              uint32_t u[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                u[e] = pack_bf16(__uint_as_float(w[q * 8 + 2 * e]) * p.scale,
                                 __uint_as_float(w[q * 8 + 2 * e + 1]) * p.scale);
              *reinterpret_cast<uint4*>(row + c * 32 + q * 8) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ------------------------------------------------------------------ dK, dV
constexpr int KV_QUERIES = 64;
constexpr int DKV_THREADS = 64 + 512;  // TMA warp, MMA warp, two groups of 8 softmax warps

template <int DQP, int DVP>
struct DaDkvSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int BLK = DA_TILE * 128, QBLK = KV_QUERIES * 128;
  static constexpr int K_BYTES = KBQ * BLK, V_BYTES = KBV * BLK, Q_BYTES = KBQ * QBLK, DO_BYTES = KBV * QBLK;
  static constexpr int ST = 4;  // Q / dO stages
  static constexpr int VEC = 4 * KV_QUERIES;  // lse2, delta, lo, hi of a step's queries
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + K_BYTES;
  static constexpr int OFF_Q = OFF_V + V_BYTES;
  static constexpr int OFF_DO = OFF_Q + ST * Q_BYTES;
  static constexpr int OFF_VEC = OFF_DO + ST * DO_BYTES;
  static constexpr int OFF_BAR = OFF_VEC + ST * VEC * 4;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

// Where a CTA's dK, dV go: bf16 rows, or (splits > 1) f32 parts [split][B, Hk, S, Dv + Dqk]
struct DkvOut {
  __nv_bfloat16 *dk, *dv;
  int64_t ldk, ldv;
  float* part;
  int splits;
};

// Transposed tiles: TMEM lanes are keys, columns the 64 queries of a step.  TMEM: dV, dK, two buffers of S^T
// (then P^T) and of dP^T (then dS^T).  The softmax warps are two groups that take the steps in turn, each with
// its buffers: while a group works on its step the tensor cores work for the other's.  A warp owns 32 keys and
// 32 queries.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DKV_THREADS, 1)
    da_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, DaParams p,
                  const float* __restrict__ lse2, const float* __restrict__ delta, DkvOut out) {
  using L = DaDkvSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sK = smem + L::OFF_K, *sV = smem + L::OFF_V, *sQ = smem + L::OFF_Q, *sDO = smem + L::OFF_DO;
  float* s_vec = reinterpret_cast<float*>(smem + L::OFF_VEC);  // [stage][4][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* kv_full = bars + 0;
  uint64_t* q_full = bars + 1;     // [4] Q, dO tiles
  uint64_t* q_empty = bars + 5;    // [4]
  uint64_t* vec_full = bars + 9;   // [4] the step's vectors
  uint64_t* s_full = bars + 13;    // [2] per buffer
  uint64_t* dp_full = bars + 15;   // [2]
  uint64_t* p_full = bars + 17;    // [2]
  uint64_t* ds_full = bars + 19;   // [2]
  uint64_t* all_done = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  // the first key tiles have the most (causal) queries and start first
  const int kt = blockIdx.z, hk = blockIdx.x / out.splits, part = blockIdx.x % out.splits, b = blockIdx.y;
  const int group = p.Hq / p.Hk;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < L::ST; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&vec_full[i], 32);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&dp_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&ds_full[i], 8);
    }
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  // this CTA's share of the (query head, 64 queries) steps that see the key tile
  TileRange qr = query_tiles(p, b, kt);
  qr.begin *= 2;
  qr.end = min(qr.end * 2, (p.S + KV_QUERIES - 1) / KV_QUERIES);
  const int ni = max(qr.end - qr.begin, 0), total = group * ni;
  const int first = (int)((int64_t)total * part / out.splits), n = (int)((int64_t)total * (part + 1) / out.splits) - first;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t TM_DV = tmem, TM_DK = tmem + 128, TM_S = tmem + 256, TM_DP = tmem + 384;

  if (warp == 0) {
    if (n > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(kv_full, L::K_BYTES + L::V_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sK + kb * L::BLK, &tmK, kv_full, kb * 64, hk, kt * DA_TILE, b);
#pragma unroll
        for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sV + kb * L::BLK, &tmV, kv_full, kb * 64, hk, kt * DA_TILE, b);
      }
      int h = hk * group + first / ni, qi = first % ni;
      int it = 0;
      for (; it < n; ++it) {
        const int st = it % L::ST;
        const int q0 = (qr.begin + qi) * KV_QUERIES;
        if (!warp_wait(&q_empty[st], ((it / L::ST) & 1) ^ 1, abort_flag, p.status)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[st], L::Q_BYTES + L::DO_BYTES);
#pragma unroll
          for (int kb = 0; kb < L::KBQ; ++kb)
            tma_load_4d(sQ + st * L::Q_BYTES + kb * L::QBLK, &tmQ, &q_full[st], kb * 64, h, q0, b);
#pragma unroll
          for (int kb = 0; kb < L::KBV; ++kb)
            tma_load_4d(sDO + st * L::DO_BYTES + kb * L::QBLK, &tmDO, &q_full[st], kb * 64, h, q0, b);
        }
        float* vec = s_vec + st * L::VEC;
        const int64_t base = ((int64_t)b * p.Hq + h) * p.S;
#pragma unroll
        for (int c = 0; c < KV_QUERIES / 32; ++c) {
          const int q = c * 32 + lane, qpos = q0 + q;
          const bool in = qpos < p.S;
          const TileRange v = key_range(p, b, qpos);
          vec[q] = in ? __ldg(lse2 + base + qpos) : INFINITY;
          vec[KV_QUERIES + q] = in ? __ldg(delta + base + qpos) : 0.f;
          reinterpret_cast<int*>(vec)[2 * KV_QUERIES + q] = v.begin;
          reinterpret_cast<int*>(vec)[3 * KV_QUERIES + q] = v.end;
        }
        mbar_arrive(&vec_full[st]);
        if (++qi == ni) {
          qi = 0;
          ++h;
        }
      }
      if (lane == 0) {
        mbar_wait(kv_full, 0, nullptr, p.status);
        for (int u = max(0, it - L::ST); u < it; ++u) mbar_wait(&q_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t lead = elect_lead();
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, KV_QUERIES, false, false);
      constexpr uint32_t ID_V = umma_idesc_bf16(DA_TILE, DVP, false, true);
      constexpr uint32_t ID_K = umma_idesc_bf16(DA_TILE, DQP, false, true);
      const int nkq = (p.Dqk + 15) / 16, nkv = (p.Dv + 15) / 16;
      const DaDesc dK = da_desc(smem_u32(sK), 16), dV = da_desc(smem_u32(sV), 16);
      bool ok = warp_wait(kv_full, 0, abort_flag, p.status);
      auto a_q = [&](int it) { return smem_u32(sQ + (it % L::ST) * L::Q_BYTES); };
      auto a_do = [&](int it) { return smem_u32(sDO + (it % L::ST) * L::DO_BYTES); };
      // S^T over P^T of two steps before, dP^T over its dS^T: both read by products issued before
      auto issue_s = [&](int it) -> bool {
        if (!warp_wait(&q_full[it % L::ST], (it / L::ST) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        da_mma_kk<DQP, L::BLK, L::QBLK>(lead, TM_S + (it & 1) * KV_QUERIES, dK, da_desc(a_q(it), 16), ID_S, nkq);
        da_commit(lead, &s_full[it & 1]);
        return true;
      };
      auto issue_dp = [&](int it) {
        da_mma_kk<DVP, L::BLK, L::QBLK>(lead, TM_DP + (it & 1) * KV_QUERIES, dV, da_desc(a_do(it), 16), ID_S, nkv);
        da_commit(lead, &dp_full[it & 1]);
      };
      // queries 16 kk ..: 32 queries a softmax warp, as bf16 in the first half of its columns
      auto a_t = [&](uint32_t t, int it, int kk) { return t + (it & 1) * KV_QUERIES + (kk >> 1) * 32 + (kk & 1) * 8; };
      for (int it = 0; it < 2 && it < n && ok; ++it) {
        ok = issue_s(it);
        if (ok) issue_dp(it);
      }
      for (int it = 0; it < n && ok; ++it) {
        if (!warp_wait(&p_full[it & 1], (it >> 1) & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const DaDesc dDO = da_desc(a_do(it), L::QBLK), dQ = da_desc(a_q(it), L::QBLK);
#pragma unroll
        for (int kk = 0; kk < KV_QUERIES / 16; ++kk)
          da_mma_ts(lead, TM_DV, a_t(TM_S, it, kk), dDO.at(kk * 2048), ID_V,
                    (it | kk) != 0);
        if (it + 2 < n && !issue_s(it + 2)) { ok = false; break; }
        if (!warp_wait(&ds_full[it & 1], (it >> 1) & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < KV_QUERIES / 16; ++kk)
          da_mma_ts(lead, TM_DK, a_t(TM_DP, it, kk), dQ.at(kk * 2048), ID_K,
                    (it | kk) != 0);
        da_commit(lead, &q_empty[it % L::ST]);
        if (it + 2 < n) issue_dp(it + 2);
        if (it + 1 == n) da_commit(lead, all_done);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, sub = (warp - 2) >> 2;  // 32 keys; half a group (or an output column block)
    const int mine = sub >> 1, half = sub & 1;            // group, 32 queries
    const int r = quarter * 32 + lane;
    const int kpos = kt * DA_TILE + r;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = TM_S + mine * KV_QUERIES + lane_base + half * 32;
    const uint32_t dp_addr = TM_DP + mine * KV_QUERIES + lane_base + half * 32;
    const float C = ALIBI ? 1.f : p.c_log2;
    bool ok = true;
    int h = 0, qi = 0;
    if (n > mine) {
      h = hk * group + (first + mine) / ni;
      qi = (first + mine) % ni;
    }
    for (int it = mine; it < n; it += 2) {
      const int st = it % L::ST, u = it / L::ST, ph = (it >> 1) & 1;
      const int q0 = (qr.begin + qi) * KV_QUERIES;
      // every query of the step sees every key of this warp?
      bool masked;
      bool padded = false;
      if (p.qt) {
        const int4 t = __ldg(p.qt + (int64_t)b * p.nt + q0 / DA_TILE);
        const int w0 = kt * DA_TILE + quarter * 32;
        masked = !(t.z <= w0 && w0 + 32 <= t.w) || q0 + KV_QUERIES > p.S;
        padded = t.z == INT_MAX;
      } else {
        masked = (p.causal && q0 < kt * DA_TILE + DA_TILE) || kt * DA_TILE + DA_TILE > p.S || q0 + KV_QUERIES > p.S;
      }
      const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
      qi += 2;
      while (qi >= ni) {
        qi -= ni;
        ++h;
      }
      const float4* vec = reinterpret_cast<const float4*>(s_vec + st * L::VEC + half * 32);
      const int4* ivec = reinterpret_cast<const int4*>(vec);
      const float fd = (float)(q0 + half * 32 - kpos);
      if (!mbar_wait(&vec_full[st], u & 1, abort_flag, p.status) ||
          !mbar_wait(&s_full[mine], ph, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[32], pk[16];
      tmem_ld32(s_addr, x);
      tc_wait_ld();
      // x becomes P times the cap's derivative, pk P
      auto probabilities = [&](auto near) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l4 = vec[e / 4];
          const float ls[4] = {l4.x, l4.y, l4.z, l4.w};
          float pr[4], w[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v = __uint_as_float(x[e + g]);
            w[g] = 1.f;
            if (CAP) v = tanh_score<decltype(near)::value>(v * p.x_scale, w[g]);
            if (ALIBI) v = fmaf(-slope2, fabsf(fd + (float)(e + g)), v * p.c_log2);
            pr[g] = ex2_approx(fmaf(v, C, -ls[g]));
            w[g] = CAP ? pr[g] * w[g] : pr[g];
          }
          if (masked) {
            const int4 lo = ivec[2 * KV_QUERIES / 4 + e / 4], hi = ivec[3 * KV_QUERIES / 4 + e / 4];
            const int lo4[4] = {lo.x, lo.y, lo.z, lo.w}, hi4[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const bool sees = lo4[g] <= kpos && kpos < hi4[g];
              pr[g] = sees ? pr[g] : 0.f;
              w[g] = sees ? w[g] : 0.f;  // the score of a hidden pair may be NaN
            }
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) x[e + g] = __float_as_uint(w[g]);
          pk[e / 2] = pack_bf16(pr[0], pr[1]);
          pk[e / 2 + 1] = pack_bf16(pr[2], pr[3]);
        }
      };
      if (CAP && warp_near<32>(x, p.x_scale)) probabilities(std::true_type{});
      else probabilities(std::false_type{});
      tmem_st16(s_addr, pk);
      if (padded) {
        if (!mbar_wait(&q_full[st], u & 1, abort_flag, p.status)) { ok = false; break; }
        zero_pad_rows<L::KBV, KV_QUERIES>(sDO + st * L::DO_BYTES, p, b, q0, half * 128 + r, 256);
        zero_pad_rows<L::KBQ, KV_QUERIES>(sQ + st * L::Q_BYTES, p, b, q0, half * 128 + r, 256);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[mine]);
      if (!mbar_wait(&dp_full[mine], ph, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t d[32];
      tmem_ld32(dp_addr, d);
      tc_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 d4 = vec[KV_QUERIES / 4 + e / 4];
        const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
        float ds[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float w = __uint_as_float(x[e + g]);
          ds[g] = w * (__uint_as_float(d[e + g]) - dl[g]);
          if (masked) ds[g] = w == 0.f ? 0.f : ds[g];  // a hidden pair adds nothing, whatever dP is
        }
        pk[e / 2] = pack_bf16(ds[0], ds[1]);
        pk[e / 2 + 1] = pack_bf16(ds[2], ds[3]);
      }
      tmem_st16(dp_addr, pk);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[mine]);
    }
    if (ok && n > 0 && !mbar_wait(all_done, 0, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const int width = which ? p.Dqk : p.Dv;
        const float f = which ? p.scale : 1.f;
        const uint32_t src = (which ? TM_DK : TM_DV) + lane_base;
#pragma unroll 1
        for (int c = sub; c < (which ? DQP : DVP) / 32; c += 4) {
          uint32_t w[32];
          if (n > 0) {
            tmem_ld32(src + c * 32, w);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = 0u;
          }
          if (kpos >= p.S) continue;
          if (out.splits > 1) {
            float* row = out.part + ((((int64_t)part * p.B + b) * p.Hk + hk) * p.S + kpos) * (p.Dqk + p.Dv) +
                         (which ? p.Dv : 0) + c * 32;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (c * 32 + q * 4 < width)
                *reinterpret_cast<float4*>(row + q * 4) =
                    make_float4(__uint_as_float(w[q * 4]) * f, __uint_as_float(w[q * 4 + 1]) * f,
                                __uint_as_float(w[q * 4 + 2]) * f, __uint_as_float(w[q * 4 + 3]) * f);
          } else {
            __nv_bfloat16* row = which ? out.dk + ((int64_t)b * p.S + kpos) * out.ldk + (int64_t)hk * p.Dqk
                                       : out.dv + ((int64_t)b * p.S + kpos) * out.ldv + (int64_t)hk * p.Dv;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (c * 32 + q * 8 < width) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  o[e] = pack_bf16(__uint_as_float(w[q * 8 + 2 * e]) * f, __uint_as_float(w[q * 8 + 2 * e + 1]) * f);
                *reinterpret_cast<uint4*>(row + c * 32 + q * 8) = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dK, dV = the splits' parts added in order; 8 columns a thread
__global__ void __launch_bounds__(256) da_join_kernel(const float* __restrict__ part, int splits, int B, int S, int Hk,
                                                      int Dqk, int Dv, __nv_bfloat16* __restrict__ dk, int64_t ldk,
                                                      __nv_bfloat16* __restrict__ dv, int64_t ldv) {
  const int vec = (Dqk + Dv) / 8;
  const int64_t total = (int64_t)B * Hk * S * vec;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int c = (int)(i % vec) * 8;
    const int64_t row = i / vec, s = row % S, bh = row / S, h = bh % Hk, b = bh / Hk;
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < splits; ++q) {
      const float4* src = reinterpret_cast<const float4*>(part + ((int64_t)q * B * Hk * S + row) * (Dqk + Dv) + c);
      const float4 x = __ldg(src), y = __ldg(src + 1);
      a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w;
      a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
    }
    __nv_bfloat16* dst = c < Dv ? dv + (b * S + s) * ldv + h * Dv + c : dk + (b * S + s) * ldk + h * Dqk + (c - Dv);
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(a[4], a[5]),
                                                pack_bf16(a[6], a[7]));
  }
}

struct BwdArgs {
  DaShape s;
  DaTensor q, k, v, o, dout;
  const float* lse2;
  float *delta, *part;
  DaOut dq, dk, dv;
  int* status;
  cudaStream_t st;
};

template <int DQP, int DVP, bool CAP, bool ALIBI>
void launch_bwd_t(const BwdArgs& a) {
  const DaShape& s = a.s;
  const CUtensorMap tq = da_tmap(a.q, s.B, s.S, s.Hq, s.Dqk), td = da_tmap(a.dout, s.B, s.S, s.Hq, s.Dv),
                    tk = da_tmap(a.k, s.B, s.S, s.Hk, s.Dqk), tv = da_tmap(a.v, s.B, s.S, s.Hk, s.Dv),
                    tk64 = da_tmap(a.k, s.B, s.S, s.Hk, s.Dqk, DQ_KEYS), tv64 = da_tmap(a.v, s.B, s.S, s.Hk, s.Dv, DQ_KEYS),
                    tq64 = da_tmap(a.q, s.B, s.S, s.Hq, s.Dqk, KV_QUERIES), td64 = da_tmap(a.dout, s.B, s.S, s.Hq, s.Dv, KV_QUERIES);
  const DaParams p = da_params(s, a.status);
  auto kq = da_dq_kernel<DQP, DVP, CAP, ALIBI>;
  auto kkv = da_dkv_kernel<DQP, DVP, CAP, ALIBI>;
  da_smem(kq, DaDqSmem<DQP, DVP>::TOTAL);
  da_smem(kkv, DaDkvSmem<DQP, DVP>::TOTAL);
  kq<<<dim3(s.Hq, s.B, p.nt), DQ_THREADS, DaDqSmem<DQP, DVP>::TOTAL, a.st>>>(
      tq, tk64, tv64, td, p, a.o, a.dout, a.lse2, a.delta, reinterpret_cast<__nv_bfloat16*>(a.dq.ptr), a.dq.ld);
  OXI_CUDA_CHECK(cudaGetLastError());
  DkvOut out;
  out.dk = reinterpret_cast<__nv_bfloat16*>(a.dk.ptr);
  out.dv = reinterpret_cast<__nv_bfloat16*>(a.dv.ptr);
  out.ldk = a.dk.ld;
  out.ldv = a.dv.ld;
  out.part = a.part;
  out.splits = da_bwd_splits(s.B, s.S, s.Hq, s.Hk);
  kkv<<<dim3(s.Hk * out.splits, s.B, p.nt), DKV_THREADS, DaDkvSmem<DQP, DVP>::TOTAL, a.st>>>(tq64, tk, tv, td64, p, a.lse2,
                                                                                             a.delta, out);
  OXI_CUDA_CHECK(cudaGetLastError());
  if (out.splits > 1) {
    const int64_t threads = (int64_t)s.B * s.Hk * s.S * ((s.Dqk + s.Dv) / 8);
    da_join_kernel<<<(unsigned)std::min<int64_t>((threads + 255) / 256, 148 * 16), 256, 0, a.st>>>(
        a.part, out.splits, s.B, s.S, s.Hk, s.Dqk, s.Dv, out.dk, out.ldk, out.dv, out.ldv);
    OXI_CUDA_CHECK(cudaGetLastError());
  }
}

template <int DQP, int DVP>
void launch_bwd_d(const BwdArgs& a) {
  if (a.s.cap > 0.f) a.s.slopes ? launch_bwd_t<DQP, DVP, true, true>(a) : launch_bwd_t<DQP, DVP, true, false>(a);
  else a.s.slopes ? launch_bwd_t<DQP, DVP, false, true>(a) : launch_bwd_t<DQP, DVP, false, false>(a);
}

}  // namespace

// A key tile's CTA walks every query head of its group: with few key heads and rows the CTAs are few
// and, under causality, as unequal as can be.  Then each tile's work is cut into parts of its own.
int da_bwd_splits(int B, int S, int Hq, int Hk) {
  const int64_t tiles = (S + DA_TILE - 1) / DA_TILE, ctas = tiles * B * Hk, most = tiles * (Hq / Hk);
  if (ctas >= 2 * 148 || most < 8) return 1;
  return (int)std::min<int64_t>(std::min<int64_t>((4 * 148 + ctas - 1) / ctas, most / 4), 8);
}

void launch_da_bwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaTensor& o,
                   const DaTensor& dout, const float* lse2, float* delta, float* part, const DaOut& dq, const DaOut& dk,
                   const DaOut& dv, int* status, cudaStream_t st) {
  if (s.B == 0 || s.S == 0 || s.Hq == 0) return;
  da_check(s);
  for (const DaOut* t : {&dq, &dk, &dv})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->ld % 8 == 0, "16-byte aligned gradient rows");
  for (const DaTensor* t : {&o, &dout})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->sb % 8 == 0 && t->ss % 8 == 0 && t->sh % 8 == 0,
              "16-byte aligned rows of the output and its gradient");
  OXI_CHECK(da_bwd_splits(s.B, s.S, s.Hq, s.Hk) == 1 || part != nullptr, "attention backward needs its parts' workspace");
  const BwdArgs a{s, q, k, v, o, dout, lse2, delta, part, dq, dk, dv, status, st};
  if (s.Dqk <= 64 && s.Dv <= 64) launch_bwd_d<64, 64>(a);
  else if (s.Dv <= 64) launch_bwd_d<128, 64>(a);
  else launch_bwd_d<128, 128>(a);
}

}  // namespace oxi
