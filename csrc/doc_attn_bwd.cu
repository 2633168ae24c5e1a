// Attention over visible key ranges for sm_100a (tcgen05 + TMEM + TMA), backward.
//
//   P  = 2^(a log2 e - lse2),  dP = dO V^T,  dS = P (dP - delta) (1 - (u / cap)^2),  delta_i = dO_i . o_i
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels that each own their outputs, so no gradient is summed with atomics and the results do
// not depend on the order in which CTAs run; each recomputes S and dP (seven tile products where one
// kernel with an atomic dQ has five):
//   dQ:     one CTA per (128 queries, query head, batch), over key tiles
//   dK, dV: one CTA per (128 keys, key head, batch), over the query heads of the group and query tiles
// Both keep their accumulators in TMEM and feed dS (and P^T) to the tensor cores from TMEM, written by
// the softmax warps over the scores they were computed from.
#include "doc_attn.cuh"

namespace oxi {
namespace {

// ------------------------------------------------------------------ delta
// delta[b, h, s] = sum_d dO o, one warp per 32 / (Dv / 8) rows: every thread reads 16 bytes of each.
__global__ void __launch_bounds__(256) da_delta_kernel(const __nv_bfloat16* __restrict__ o, int64_t osb, int64_t oss,
                                                       int64_t osh, const __nv_bfloat16* __restrict__ d, int64_t dsb,
                                                       int64_t dss, int64_t dsh, int B, int S, int Hq, int Dv,
                                                       float* __restrict__ delta) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)B * S * Hq;
  for (int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; row < rows; row += (int64_t)gridDim.x * 8) {
    const int h = (int)(row % Hq);
    const int64_t t = row / Hq, b = t / S, s = t % S;
    float sum = 0.f;
    if (lane * 8 < Dv) {
      const uint4 x = *reinterpret_cast<const uint4*>(o + b * osb + s * oss + h * osh + lane * 8);
      const uint4 y = *reinterpret_cast<const uint4*>(d + b * dsb + s * dss + h * dsh + lane * 8);
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack_bf16(xw[i]), c = unpack_bf16(yw[i]);
        sum = fmaf(a.x, c.x, fmaf(a.y, c.y, sum));
      }
    }
#pragma unroll
    for (int q = 8; q > 0; q >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, q);
    if (lane == 0) delta[(b * Hq + h) * S + s] = sum;
  }
}

// ------------------------------------------------------------------ dQ
template <int DQP, int DVP>
struct DaDqSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int BLK = DA_TILE * 128;
  static constexpr int Q_BYTES = KBQ * BLK, V_BYTES = KBV * BLK;
  static constexpr int ST = 2;  // K / V stages
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_DO = OFF_Q + Q_BYTES;
  static constexpr int OFF_K = OFF_DO + V_BYTES;
  static constexpr int OFF_V = OFF_K + ST * Q_BYTES;
  static constexpr int OFF_BAR = OFF_V + ST * V_BYTES;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

// One column half (64 keys) of a 128 x 128 tile per warp, 32 query rows; TMEM: dQ, two S buffers, dP.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DA_THREADS, 1)
    da_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, DaParams p,
                 const float* __restrict__ lse2, const float* __restrict__ delta, __nv_bfloat16* __restrict__ dq,
                 int64_t ld) {
  using L = DaDqSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem + L::OFF_Q, *sDO = smem + L::OFF_DO, *sK = smem + L::OFF_K, *sV = smem + L::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* kv_full = bars + 1;   // [2]
  uint64_t* kv_empty = bars + 3;  // [2]
  uint64_t* s_full = bars + 5;    // S and dP of a key tile
  uint64_t* dp_free = bars + 6;   // dP has been read into registers
  uint64_t* ds_full = bars + 7;
  uint64_t* all_done = bars + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 9);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int qt = gridDim.z - 1 - blockIdx.z, h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (p.Hq / p.Hk);
  const TileRange kr = key_tiles(p, b, qt);
  const int n = kr.end - kr.begin;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_free, 8);
    mbar_init(ds_full, 8);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t TM_DQ = tmem, TM_S = tmem + 128, TM_DP = tmem + 384;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_full, L::Q_BYTES + L::V_BYTES);
#pragma unroll
      for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sQ + kb * L::BLK, &tmQ, q_full, kb * 64, h, qt * DA_TILE, b);
#pragma unroll
      for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sDO + kb * L::BLK, &tmDO, q_full, kb * 64, h, qt * DA_TILE, b);
      int i = 0;
      for (; i < n; ++i) {
        const int st = i % L::ST;
        if (!mbar_wait(&kv_empty[st], ((i / L::ST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(&kv_full[st], L::Q_BYTES + L::V_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sK + st * L::Q_BYTES + kb * L::BLK, &tmK, &kv_full[st], kb * 64, hk, (kr.begin + i) * DA_TILE, b);
#pragma unroll
        for (int kb = 0; kb < L::KBV; ++kb)
          tma_load_4d(sV + st * L::V_BYTES + kb * L::BLK, &tmV, &kv_full[st], kb * 64, hk, (kr.begin + i) * DA_TILE, b);
      }
      mbar_wait(q_full, 0, nullptr, p.status);
      for (int u = max(0, i - L::ST); u < i; ++u) mbar_wait(&kv_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, DA_TILE, false, false);
      constexpr uint32_t ID_Q = umma_idesc_bf16(DA_TILE, DQP, false, true);
      const int nkq = (p.Dqk + 15) / 16, nkv = (p.Dv + 15) / 16;
      const uint32_t aQ = smem_u32(sQ), aDO = smem_u32(sDO);
      bool ok = mbar_wait(q_full, 0, abort_flag, p.status);
      // S_i into buffer i & 1, which last held dS_{i-2}, read by a product issued before; dP_i once
      // the softmax warps have read dP_{i-1}
      auto issue = [&](int i) -> bool {
        const int st = i % L::ST;
        if (!mbar_wait(&kv_full[st], (i / L::ST) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        const uint32_t aK = smem_u32(sK + st * L::Q_BYTES), aV = smem_u32(sV + st * L::V_BYTES);
        for (int kk = 0; kk < nkq; ++kk)
          tc_mma_f16(TM_S + (i & 1) * 128, da_kmajor_desc(aQ, kk, L::BLK), da_kmajor_desc(aK, kk, L::BLK), ID_S, kk != 0);
        if (i > 0 && !mbar_wait(dp_free, (i - 1) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        for (int kk = 0; kk < nkv; ++kk)
          tc_mma_f16(TM_DP, da_kmajor_desc(aDO, kk, L::BLK), da_kmajor_desc(aV, kk, L::BLK), ID_S, kk != 0);
        tc_commit(s_full);
        return true;
      };
      if (ok) ok = issue(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && !issue(i + 1)) { ok = false; break; }
        if (!mbar_wait(ds_full, i & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t aK = smem_u32(sK + (i % L::ST) * L::Q_BYTES);
#pragma unroll
        for (int kk = 0; kk < DA_TILE / 16; ++kk)  // keys 0..63 in columns 0..31, 64..127 in columns 64..95
          tc_mma_f16_ts(TM_DQ, TM_S + (i & 1) * 128 + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8),
                        umma_desc_sw128(aK + kk * 2048, L::BLK, 1024), ID_Q, (i | kk) != 0);
        tc_commit(&kv_empty[i % L::ST]);
        if (i == n - 1) tc_commit(all_done);
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
    const int64_t vi = ((int64_t)b * p.Hq + h) * p.S + qpos;
    const float ls = qpos < p.S ? lse2[vi] : INFINITY, dl = qpos < p.S ? delta[vi] : 0.f;
    const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
    const float C = ALIBI ? 1.f : p.c_log2;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int k0 = (kr.begin + i) * DA_TILE + half * 64;
      if (!mbar_wait(s_full, i & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      const uint32_t s_addr = TM_S + (i & 1) * 128 + lane_base + half * 64;
      uint32_t x[2][32], d[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tmem_ld32(s_addr + c * 32, x[c]);
        tmem_ld32(TM_DP + lane_base + half * 64 + c * 32, d[c]);
      }
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_free);
      const bool masked = !(all_lo <= k0 && k0 + 64 <= all_hi);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float fd = (float)(qpos - (k0 + c * 32));
        const uint32_t bits = masked ? range_bits(vis.begin, vis.end, k0 + c * 32) : 0xffffffffu;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float v = __uint_as_float(x[c][e]), f = 1.f;
          if (CAP) v = tanh_ex2(v * p.x_scale, f);
          if (ALIBI) v = fmaf(-slope2, fabsf(fd - (float)e), v * p.c_log2);
          float ds = ex2_approx(fmaf(v, C, -ls)) * (__uint_as_float(d[c][e]) - dl);
          if (CAP) ds *= f;
          x[c][e] = __float_as_uint(ds);
        }
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((bits >> e) & 1u)) x[c][e] = 0u;
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack_bf16(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1]));
        tmem_st16(s_addr + c * 16, pk);
      }
      // S_i has read K_i: rows of padding become zero before the dQ product reads them
      if (tile_has_pad(p, b, kr.begin + i))
        zero_pad_rows<L::KBQ>(sK + (i % L::ST) * L::Q_BYTES, p, b, (kr.begin + i) * DA_TILE, half * 128 + r, 256);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && n > 0 && !mbar_wait(all_done, 0, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
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
        if (qpos < p.S) {
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
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ dK, dV
template <int DQP, int DVP>
struct DaDkvSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int BLK = DA_TILE * 128;
  static constexpr int Q_BYTES = KBQ * BLK, V_BYTES = KBV * BLK;
  static constexpr int ST = 2;  // Q / dO stages
  static constexpr int VEC_BYTES = 4 * DA_TILE * 4;  // lse2, delta, lo, hi of a query tile
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + Q_BYTES;
  static constexpr int OFF_Q = OFF_V + V_BYTES;
  static constexpr int OFF_DO = OFF_Q + ST * Q_BYTES;
  static constexpr int OFF_VEC = OFF_DO + ST * V_BYTES;
  static constexpr int OFF_BAR = OFF_VEC + ST * VEC_BYTES;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

// Transposed tiles: TMEM lanes are keys, columns queries.  TMEM: dV, dK, S^T (then P^T), dP^T (then dS^T).
// A warp owns 32 keys and 64 of the tile's queries.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DA_THREADS, 1)
    da_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, DaParams p,
                  const float* __restrict__ lse2, const float* __restrict__ delta, __nv_bfloat16* __restrict__ dk,
                  int64_t ldk, __nv_bfloat16* __restrict__ dv, int64_t ldv) {
  using L = DaDkvSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sK = smem + L::OFF_K, *sV = smem + L::OFF_V, *sQ = smem + L::OFF_Q, *sDO = smem + L::OFF_DO;
  float* s_vec = reinterpret_cast<float*>(smem + L::OFF_VEC);  // [stage][4][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* kv_full = bars + 0;
  uint64_t* q_full = bars + 1;     // [2] Q, dO tiles
  uint64_t* q_empty = bars + 3;    // [2]
  uint64_t* vec_full = bars + 5;   // [2] the tile's vectors
  uint64_t* s_full = bars + 7;
  uint64_t* dp_full = bars + 8;
  uint64_t* p_full = bars + 9;
  uint64_t* ds_full = bars + 10;
  uint64_t* all_done = bars + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // the first key tiles have the most (causal) queries and start first
  const int kt = blockIdx.z, hk = blockIdx.x, b = blockIdx.y;
  const int group = p.Hq / p.Hk;
  const TileRange qr = query_tiles(p, b, kt);
  const int ni = qr.end - qr.begin, n = group * ni;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&vec_full[i], 32);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 8);
    mbar_init(ds_full, 8);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t TM_DV = tmem, TM_DK = tmem + 128, TM_S = tmem + 256, TM_DP = tmem + 384;

  if (warp == 0) {
    if (n > 0) {
      if (lane == 0) {
        mbar_arrive_expect_tx(kv_full, L::Q_BYTES + L::V_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sK + kb * L::BLK, &tmK, kv_full, kb * 64, hk, kt * DA_TILE, b);
#pragma unroll
        for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sV + kb * L::BLK, &tmV, kv_full, kb * 64, hk, kt * DA_TILE, b);
      }
      int it = 0;
      for (; it < n; ++it) {
        const int st = it % L::ST;
        const int h = hk * group + it / ni, q0 = (qr.begin + it % ni) * DA_TILE;
        const bool ok = mbar_wait(&q_empty[st], ((it / L::ST) & 1) ^ 1, abort_flag, p.status);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[st], L::Q_BYTES + L::V_BYTES);
#pragma unroll
          for (int kb = 0; kb < L::KBQ; ++kb)
            tma_load_4d(sQ + st * L::Q_BYTES + kb * L::BLK, &tmQ, &q_full[st], kb * 64, h, q0, b);
#pragma unroll
          for (int kb = 0; kb < L::KBV; ++kb)
            tma_load_4d(sDO + st * L::V_BYTES + kb * L::BLK, &tmDO, &q_full[st], kb * 64, h, q0, b);
        }
        float* vec = s_vec + st * 4 * DA_TILE;
        const int64_t base = ((int64_t)b * p.Hq + h) * p.S;
#pragma unroll
        for (int c = 0; c < DA_TILE / 32; ++c) {
          const int q = c * 32 + lane, qpos = q0 + q;
          const bool in = qpos < p.S;
          const TileRange v = key_range(p, b, qpos);
          vec[q] = in ? __ldg(lse2 + base + qpos) : INFINITY;
          vec[DA_TILE + q] = in ? __ldg(delta + base + qpos) : 0.f;
          reinterpret_cast<int*>(vec)[2 * DA_TILE + q] = v.begin;
          reinterpret_cast<int*>(vec)[3 * DA_TILE + q] = v.end;
        }
        mbar_arrive(&vec_full[st]);
      }
      if (lane == 0) {
        mbar_wait(kv_full, 0, nullptr, p.status);
        for (int u = max(0, it - L::ST); u < it; ++u) mbar_wait(&q_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, DA_TILE, false, false);
      constexpr uint32_t ID_V = umma_idesc_bf16(DA_TILE, DVP, false, true);
      constexpr uint32_t ID_K = umma_idesc_bf16(DA_TILE, DQP, false, true);
      const int nkq = (p.Dqk + 15) / 16, nkv = (p.Dv + 15) / 16;
      const uint32_t aK = smem_u32(sK), aV = smem_u32(sV);
      bool ok = mbar_wait(kv_full, 0, abort_flag, p.status);
      auto a_q = [&](int it) { return smem_u32(sQ + (it % L::ST) * L::Q_BYTES); };
      auto a_do = [&](int it) { return smem_u32(sDO + (it % L::ST) * L::V_BYTES); };
      // S^T over P^T of the pair before, dP^T over its dS^T: both read by products issued before
      auto issue_s = [&](int it) {
        for (int kk = 0; kk < nkq; ++kk)
          tc_mma_f16(TM_S, da_kmajor_desc(aK, kk, L::BLK), da_kmajor_desc(a_q(it), kk, L::BLK), ID_S, kk != 0);
        tc_commit(s_full);
      };
      auto issue_dp = [&](int it) {
        for (int kk = 0; kk < nkv; ++kk)
          tc_mma_f16(TM_DP, da_kmajor_desc(aV, kk, L::BLK), da_kmajor_desc(a_do(it), kk, L::BLK), ID_S, kk != 0);
        tc_commit(dp_full);
      };
      auto wait_q = [&](int it) { return mbar_wait(&q_full[it % L::ST], (it / L::ST) & 1, abort_flag, p.status); };
      if (ok) ok = wait_q(0);
      if (ok) {
        tc_fence_after();
        issue_s(0);
        issue_dp(0);
      }
      for (int it = 0; it < n && ok; ++it) {
        if (!mbar_wait(p_full, it & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < DA_TILE / 16; ++kk)  // queries 0..63 in columns 0..31, 64..127 in columns 64..95
          tc_mma_f16_ts(TM_DV, TM_S + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8),
                        umma_desc_sw128(a_do(it) + kk * 2048, L::BLK, 1024), ID_V, (it | kk) != 0);
        if (it + 1 < n) {
          if (!wait_q(it + 1)) { ok = false; break; }
          tc_fence_after();
          issue_s(it + 1);
        }
        if (!mbar_wait(ds_full, it & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < DA_TILE / 16; ++kk)
          tc_mma_f16_ts(TM_DK, TM_DP + (kk < 4 ? kk * 8 : 64 + (kk - 4) * 8),
                        umma_desc_sw128(a_q(it) + kk * 2048, L::BLK, 1024), ID_K, (it | kk) != 0);
        tc_commit(&q_empty[it % L::ST]);
        if (it + 1 < n) issue_dp(it + 1);
        else tc_commit(all_done);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int r = quarter * 32 + lane;
    const int kpos = kt * DA_TILE + r;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float C = ALIBI ? 1.f : p.c_log2;
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int st = it % L::ST, u = it / L::ST;
      const int h = hk * group + it / ni, qi = qr.begin + it % ni, q0 = qi * DA_TILE;
      // every query of the tile sees every key of this warp?
      bool masked;
      bool padded = false;
      if (p.qt) {
        const int4 t = __ldg(p.qt + (int64_t)b * p.nt + qi);
        const int w0 = kt * DA_TILE + quarter * 32;
        masked = !(t.z <= w0 && w0 + 32 <= t.w) || q0 + DA_TILE > p.S;
        padded = t.z == INT_MAX;
      } else {
        masked = (p.causal && q0 < kt * DA_TILE + DA_TILE) || kt * DA_TILE + DA_TILE > p.S || q0 + DA_TILE > p.S;
      }
      const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
      const float* vec = s_vec + st * 4 * DA_TILE + half * 64;
      const int* ivec = reinterpret_cast<const int*>(vec);
      if (!mbar_wait(&vec_full[st], u & 1, abort_flag, p.status) ||
          !mbar_wait(s_full, it & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld32(TM_S + lane_base + half * 64 + c * 32, x[c]);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float fd = (float)(q0 + half * 64 + c * 32 - kpos);
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float pr[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float v = __uint_as_float(x[c][e + g]), f = 1.f;
            if (CAP) v = tanh_ex2(v * p.x_scale, f);
            if (ALIBI) v = fmaf(-slope2, fabsf(fd + (float)(e + g)), v * p.c_log2);
            float pp = ex2_approx(fmaf(v, C, -vec[c * 32 + e + g]));
            if (masked) {
              const int q = c * 32 + e + g;
              const bool sees = ivec[2 * DA_TILE + q] <= kpos && kpos < ivec[3 * DA_TILE + q];
              pp = sees ? pp : 0.f;
              if (CAP) f = sees ? f : 0.f;  // the score of a hidden pair may be NaN
            }
            pr[g] = pp;
            x[c][e + g] = __float_as_uint(CAP ? pp * f : pp);
          }
          pk[e / 2] = pack_bf16(pr[0], pr[1]);
        }
        tmem_st16(TM_S + lane_base + half * 64 + c * 16, pk);
      }
      if (padded) {
        if (!mbar_wait(&q_full[st], u & 1, abort_flag, p.status)) { ok = false; break; }
        zero_pad_rows<L::KBV>(sDO + st * L::V_BYTES, p, b, q0, half * 128 + r, 256);
        zero_pad_rows<L::KBQ>(sQ + st * L::Q_BYTES, p, b, q0, half * 128 + r, 256);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
      if (!mbar_wait(dp_full, it & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t d[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld32(TM_DP + lane_base + half * 64 + c * 32, d[c]);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float ds[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float w = __uint_as_float(x[c][e + g]);
            ds[g] = w * (__uint_as_float(d[c][e + g]) - vec[DA_TILE + c * 32 + e + g]);
            if (masked && w == 0.f) ds[g] = 0.f;  // a hidden pair adds nothing, whatever dP is
          }
          pk[e / 2] = pack_bf16(ds[0], ds[1]);
        }
        tmem_st16(TM_DP + lane_base + half * 64 + c * 16, pk);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    if (ok && n > 0 && !mbar_wait(all_done, 0, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const int width = which ? p.Dqk : p.Dv;
        __nv_bfloat16* row = which ? dk + ((int64_t)b * p.S + kpos) * ldk + (int64_t)hk * p.Dqk
                                   : dv + ((int64_t)b * p.S + kpos) * ldv + (int64_t)hk * p.Dv;
        const float f = which ? p.scale : 1.f;
        const uint32_t src = (which ? TM_DK : TM_DV) + lane_base;
#pragma unroll 1
        for (int c = half; c < (which ? DQP : DVP) / 32; c += 2) {
          uint32_t w[32];
          if (n > 0) {
            tmem_ld32(src + c * 32, w);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = 0u;
          }
          if (kpos < p.S) {
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

struct BwdArgs {
  DaShape s;
  DaTensor q, k, v, o, dout;
  const float* lse2;
  float* delta;
  DaOut dq, dk, dv;
  int* status;
  cudaStream_t st;
};

template <int DQP, int DVP, bool CAP, bool ALIBI>
void launch_bwd_t(const BwdArgs& a) {
  const DaShape& s = a.s;
  const CUtensorMap tq = da_tmap(a.q, s.B, s.S, s.Hq, s.Dqk), tk = da_tmap(a.k, s.B, s.S, s.Hk, s.Dqk),
                    tv = da_tmap(a.v, s.B, s.S, s.Hk, s.Dv), td = da_tmap(a.dout, s.B, s.S, s.Hq, s.Dv);
  const DaParams p = da_params(s, a.status);
  auto kq = da_dq_kernel<DQP, DVP, CAP, ALIBI>;
  auto kkv = da_dkv_kernel<DQP, DVP, CAP, ALIBI>;
  da_smem(kq, DaDqSmem<DQP, DVP>::TOTAL);
  da_smem(kkv, DaDkvSmem<DQP, DVP>::TOTAL);
  kkv<<<dim3(s.Hk, s.B, p.nt), DA_THREADS, DaDkvSmem<DQP, DVP>::TOTAL, a.st>>>(
      tq, tk, tv, td, p, a.lse2, a.delta, reinterpret_cast<__nv_bfloat16*>(a.dk.ptr), a.dk.ld,
      reinterpret_cast<__nv_bfloat16*>(a.dv.ptr), a.dv.ld);
  OXI_CUDA_CHECK(cudaGetLastError());
  kq<<<dim3(s.Hq, s.B, p.nt), DA_THREADS, DaDqSmem<DQP, DVP>::TOTAL, a.st>>>(
      tq, tk, tv, td, p, a.lse2, a.delta, reinterpret_cast<__nv_bfloat16*>(a.dq.ptr), a.dq.ld);
  OXI_CUDA_CHECK(cudaGetLastError());
}

template <int DQP, int DVP>
void launch_bwd_d(const BwdArgs& a) {
  if (a.s.cap > 0.f) a.s.slopes ? launch_bwd_t<DQP, DVP, true, true>(a) : launch_bwd_t<DQP, DVP, true, false>(a);
  else a.s.slopes ? launch_bwd_t<DQP, DVP, false, true>(a) : launch_bwd_t<DQP, DVP, false, false>(a);
}

}  // namespace

void launch_da_bwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaTensor& o,
                   const DaTensor& dout, const float* lse2, float* delta, const DaOut& dq, const DaOut& dk,
                   const DaOut& dv, int* status, cudaStream_t st) {
  if (s.B == 0 || s.S == 0 || s.Hq == 0) return;
  da_check(s);
  for (const DaOut* t : {&dq, &dk, &dv})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->ld % 8 == 0, "16-byte aligned gradient rows");
  OXI_CHECK((reinterpret_cast<uintptr_t>(o.ptr) & 15) == 0 && o.sb % 8 == 0 && o.ss % 8 == 0 && o.sh % 8 == 0,
            "16-byte aligned output rows");
  const int64_t rows = (int64_t)s.B * s.S * s.Hq;
  da_delta_kernel<<<(unsigned)std::min<int64_t>((rows + 7) / 8, 148 * 16), 256, 0, st>>>(
      reinterpret_cast<const __nv_bfloat16*>(o.ptr), o.sb, o.ss, o.sh, reinterpret_cast<const __nv_bfloat16*>(dout.ptr),
      dout.sb, dout.ss, dout.sh, s.B, s.S, s.Hq, s.Dv, delta);
  OXI_CUDA_CHECK(cudaGetLastError());
  const BwdArgs a{s, q, k, v, o, dout, lse2, delta, dq, dk, dv, status, st};
  if (s.Dqk <= 64 && s.Dv <= 64) launch_bwd_d<64, 64>(a);
  else if (s.Dv <= 64) launch_bwd_d<128, 64>(a);
  else launch_bwd_d<128, 128>(a);
}

}  // namespace oxi
