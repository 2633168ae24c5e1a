// Attention over visible key ranges for sm_100a (tcgen05 + TMEM + TMA), backward.
//
//   P  = 2^(a log2 e - lse2),  dP = dO V^T,  dS = P (dP - delta) (1 - (u / cap)^2),  delta_i = dO_i . o_i
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels that each own their outputs, so no gradient is summed with atomics and the results do
// not depend on the order in which CTAs run; each recomputes S and dP (seven tile products where one
// kernel with an atomic dQ has five):
//   dQ:     one CTA per (128 queries, query head, batch), over steps of 64 keys
//   dK, dV: one CTA per (128 keys, key head, batch), over the query heads of the group and steps of 64 queries
// Both keep their accumulators in TMEM and feed dS (and P^T) to the tensor cores from TMEM, written by
// the softmax warps over the scores they were computed from.
//
// What bounds them: the products of a dQ step (128 queries x 64 keys, 128-wide heads) take 788 clocks, of a dK / dV
// step 1310 (S and dP have their A operand in shared memory there), and the softmax warps' instructions about as
// long; the two overlap through the alternating groups.  dK / dV keeps to 96 registers, which the 18 warps leave a
// thread, and spills 16 to 172 bytes for it, most under a cap.  One
// dense causal row of 8192 tokens, 16 / 4 heads of 128: dQ 369 us (1118 TFLOP/s of its own three products), dK and dV
// 481 us (1143 of its four); with a cap of 50, whose tanh and derivative are instructions, 480 and 556 us; heads of 64:
// 286 and 393 us (16 / 16 heads).  8 x 2048 tokens in documents of 700, capped: 241 and 230 us.  16 x 1024 tokens in
// documents of 300, heads of 96 and 64: 104 and 112 us, 40 % of it starts and ends of CTAs (4 of 10 us, one CTA a SM): of
// rows as short as that without a mask, many at a time, flash_attn.cu's backward is the faster one.
// Tried and no faster: dK / dV's CTAs started under dQ's last wave (a programmatic launch).
//
// P and dS are rounded to bf16 for the tensor cores (2^-8 of each term at most, with random signs over the keys of a
// row); statistics, delta and accumulators are f32.  The gradients are 0.23 to 0.24 % off in the 2-norm, where products of
// f32 and one rounding of the result to bf16 leave 0.166 %.
// delta is formed in the dQ kernel, from o.  Where one key has most of a row's weight, dP - delta is what
// two nearly equal numbers leave, so an error of delta counts many times: with o rounded to bf16, dQ was
// 0.6 % off (2-norm) for documents of a few tokens with sharp scores, where the roundings of dS and dQ make
// 0.24 %.  With o in two bf16 (o + o_lo) and the forward's mean taken with one set of weights it is 0.27 %.
// The row's sum of P (dP - delta) would be zero with the true delta: the dQ kernel adds it up as it goes,
// and the dK / dV kernel behind it gets the corrected one.
#include "doc_attn.cuh"

namespace oxi {
namespace {

// A row that sees one key has no gradient through its score.  That is exact here, not what rounding leaves: the dQ
// kernel takes its P as zero, and marks it for the dK / dV kernel with this NaN in place of delta (arithmetic
// makes no such NaN).
constexpr uint32_t LONE_KEY = 0x7fc0a5a5u;

// ------------------------------------------------------------------ dQ
constexpr int DQ_KEYS = 64;
constexpr int DA_GROUPS_THREADS = 64 + 512;  // TMA warp, MMA warp, two groups of 8 softmax warps

template <int DQP, int DVP>
struct DaDqSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int QBLK = DA_TILE * 128, KBLK = DQ_KEYS * 128;
  static constexpr int Q_BYTES = KBQ * QBLK, DO_BYTES = KBV * QBLK, K_BYTES = KBQ * KBLK, V_BYTES = KBV * KBLK;
  static constexpr int ST = 4;  // K / V stages
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_DO = OFF_Q + Q_BYTES;
  static constexpr int OFF_K = OFF_DO + DO_BYTES;
  static constexpr int OFF_V = OFF_K + ST * K_BYTES;
  static constexpr int OFF_ROW = OFF_V + ST * V_BYTES;  // delta, and what it is off by, per row: [5][128] f32
  static constexpr int OFF_BAR = OFF_ROW + 5 * DA_TILE * 4;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

// 128 rows of a K-major operand tile (COLS columns, blocks of 64) from shared memory into TMEM as the A operand of
// a product: each thread its row, half the columns.
template <int COLS>
__device__ __forceinline__ void rows_to_tmem(const uint8_t* tile, uint32_t taddr, int r, int half) {
  uint32_t w[COLS / 4];
#pragma unroll
  for (int c = 0; c < COLS / 16; ++c) {
    const int chunk = half * (COLS / 16) + c;  // 8 columns
    const uint4 v = *reinterpret_cast<const uint4*>(tile + (chunk >> 3) * (DA_TILE * 128) + r * 128 +
                                                    (((chunk & 7) ^ (r & 7)) << 4));
    w[4 * c] = v.x;
    w[4 * c + 1] = v.y;
    w[4 * c + 2] = v.z;
    w[4 * c + 3] = v.w;
  }
  if constexpr (COLS == 128) tmem_st32(taddr + half * 32, w);
  else tmem_st16(taddr + half * 16, w);
}

// TMEM: dQ, Q and dO (as A operands: read from there a 128 x 64 x 16 product takes 33 clocks, with A from shared
// memory 49), two buffers of S and of dP (then dS).  The softmax warps are two groups that take the steps of 64
// keys in turn, each with its buffers: while a group works on its step the tensor cores work for the other's.  A
// warp owns 32 queries and 32 keys.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DA_GROUPS_THREADS, 1)
    da_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                 const __grid_constant__ CUtensorMap tmDQ, DaParams p, DaTensor o_in, DaTensor olo_in,
                 const float* __restrict__ nlse2, float* __restrict__ ndelta) {
  using L = DaDqSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *sQ = smem + L::OFF_Q, *sDO = smem + L::OFF_DO, *sK = smem + L::OFF_K, *sV = smem + L::OFF_V;
  float* s_row = reinterpret_cast<float*>(smem + L::OFF_ROW);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* a_full = bars + 1;     // Q and dO are in TMEM
  uint64_t* kv_full = bars + 2;    // [4]
  uint64_t* kv_empty = bars + 6;   // [4]
  uint64_t* s_full = bars + 10;    // [2] per buffer
  uint64_t* dp_full = bars + 12;   // [2]
  uint64_t* ds_full = bars + 14;   // [2]
  uint64_t* all_done = bars + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int qt = gridDim.z - 1 - blockIdx.z, h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (p.Hq / p.Hk);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(a_full, 16);
    for (int i = 0; i < L::ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 8);
    }
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    // Q and dO at once: the rest of the start runs under their latency
    mbar_arrive_expect_tx(q_full, L::Q_BYTES + L::DO_BYTES);
#pragma unroll
    for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sQ + kb * L::QBLK, &tmQ, q_full, kb * 64, h, qt * DA_TILE, b);
#pragma unroll
    for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sDO + kb * L::QBLK, &tmDO, q_full, kb * 64, h, qt * DA_TILE, b);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  const TileRange kr = key_steps(p, b, qt, DQ_KEYS);
  const int n = kr.end - kr.begin;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t TM_DQ = tmem, TM_Q = tmem + 128, TM_DO = tmem + 192, TM_S = tmem + 256, TM_DP = tmem + 384;

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < n; ++i) {
        const int st = i % L::ST;
        if (!mbar_wait(&kv_empty[st], ((i / L::ST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(&kv_full[st], L::K_BYTES + L::V_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sK + st * L::K_BYTES + kb * L::KBLK, &tmK, &kv_full[st], kb * 64, hk, (kr.begin + i) * DQ_KEYS, b);
#pragma unroll
        for (int kb = 0; kb < L::KBV; ++kb)
          tma_load_4d(sV + st * L::V_BYTES + kb * L::KBLK, &tmV, &kv_full[st], kb * 64, hk, (kr.begin + i) * DQ_KEYS, b);
      }
      // leave no copy in flight into shared memory
      mbar_wait(q_full, 0, nullptr, p.status);
      for (int u = max(0, i - L::ST); u < i; ++u) mbar_wait(&kv_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t lead = elect_lead();
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, DQ_KEYS, false, false);
      constexpr uint32_t ID_Q = umma_idesc_bf16(DA_TILE, DQP, false, true);
      const int nkq = (p.Dqk + 15) / 16, nkv = (p.Dv + 15) / 16;
      // over S_{i-2}, which its group has read before it handed dS_{i-2} over
      auto issue_s = [&](int i) -> bool {
        if (!warp_wait(&kv_full[i % L::ST], (i / L::ST) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        const DaDesc dK = da_desc(smem_u32(sK + (i % L::ST) * L::K_BYTES), 16);
#pragma unroll
        for (int kk = 0; kk < DQP / 16; ++kk)
          if (kk < nkq)
            da_mma_ts(lead, TM_S + (i & 1) * DQ_KEYS, TM_Q + kk * 8, dK.at((kk >> 2) * L::KBLK + (kk & 3) * 32), ID_S, kk != 0);
        da_commit(lead, &s_full[i & 1]);
        return true;
      };
      // over dS_{i-2}, read by a product issued before
      auto issue_dp = [&](int i) {
        const DaDesc dV = da_desc(smem_u32(sV + (i % L::ST) * L::V_BYTES), 16);
#pragma unroll
        for (int kk = 0; kk < DVP / 16; ++kk)
          if (kk < nkv)
            da_mma_ts(lead, TM_DP + (i & 1) * DQ_KEYS, TM_DO + kk * 8, dV.at((kk >> 2) * L::KBLK + (kk & 3) * 32), ID_S, kk != 0);
        da_commit(lead, &dp_full[i & 1]);
      };
      bool ok = warp_wait(a_full, 0, abort_flag, p.status);
      for (int i = 0; i < 2 && i < n && ok; ++i) {
        ok = issue_s(i);
        if (ok) issue_dp(i);
      }
      for (int i = 0; i < n && ok; ++i) {
        if (!warp_wait(&ds_full[i & 1], (i >> 1) & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const DaDesc dK = da_desc(smem_u32(sK + (i % L::ST) * L::K_BYTES), L::KBLK);
#pragma unroll
        for (int kk = 0; kk < DQ_KEYS / 16; ++kk)  // keys 0..31 in columns 0..15, 32..63 in columns 32..47
          da_mma_ts(lead, TM_DQ, TM_DP + (i & 1) * DQ_KEYS + (kk >> 1) * 32 + (kk & 1) * 8, dK.at(kk * 2048), ID_Q,
                    (i | kk) != 0);
        da_commit(lead, &kv_empty[i % L::ST]);
        if (i + 2 < n) {
          if (!issue_s(i + 2)) { ok = false; break; }
          issue_dp(i + 2);
        }
        if (i + 1 == n) da_commit(lead, all_done);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, sub = (warp - 2) >> 2;  // 32 queries; group and half of its keys
    const int mine = sub >> 1, half = sub & 1;
    const int r = quarter * 32 + lane;
    const int qpos = qt * DA_TILE + r;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    // what a row needs from memory, all in flight together
    const TileRange vis = key_range(p, b, qpos);
    const bool in = qpos < p.S;
    const int64_t vi = ((int64_t)b * p.Hq + h) * p.S + qpos;
    const bool lone = vis.end - vis.begin == 1;
    const float nls = in && !lone ? __ldg(nlse2 + vi) : -INFINITY;
    // minus delta of 8 rows a warp, 16 bytes a lane: 2 rows at a time; dO is in shared memory
    {
      const __nv_bfloat16* op = reinterpret_cast<const __nv_bfloat16*>(o_in.ptr) + b * o_in.sb + h * o_in.sh;
      const __nv_bfloat16* lp = reinterpret_cast<const __nv_bfloat16*>(olo_in.ptr) + b * olo_in.sb + h * olo_in.sh;
      const int chunk = lane & 15, row0 = (warp - 2) * 8 + (lane >> 4);
      uint4 x[4], xl[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t pos = qt * DA_TILE + row0 + 2 * g;
        x[g] = xl[g] = make_uint4(0, 0, 0, 0);
        if (pos < p.S && chunk * 8 < p.Dv) {
          x[g] = __ldg(reinterpret_cast<const uint4*>(op + pos * o_in.ss + chunk * 8));
          xl[g] = __ldg(reinterpret_cast<const uint4*>(lp + pos * olo_in.ss + chunk * 8));
        }
      }
      if (!mbar_wait(q_full, 0, abort_flag, p.status)) ok = false;
      if (ok) {
        if (mine == 0) rows_to_tmem<DQP>(sQ, TM_Q + lane_base, r, half);
        else rows_to_tmem<DVP>(sDO, TM_DO + lane_base, r, half);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(a_full);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int row = row0 + 2 * g;
        uint4 y = make_uint4(0, 0, 0, 0);
        if (chunk < DVP / 8)
          y = *reinterpret_cast<const uint4*>(sDO + (chunk >> 3) * L::QBLK + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
        const uint32_t xw[4] = {x[g].x, x[g].y, x[g].z, x[g].w}, lw[4] = {xl[g].x, xl[g].y, xl[g].z, xl[g].w},
                       yw[4] = {y.x, y.y, y.z, y.w};
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = unpack_bf16(xw[e]), l = unpack_bf16(lw[e]), d = unpack_bf16(yw[e]);
          sum = fmaf(a.x + l.x, d.x, fmaf(a.y + l.y, d.y, sum));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (chunk == 0) s_row[row] = -sum;
      }
    }
    asm volatile("bar.sync 1, 512;" ::: "memory");  // delta's rows; reached by every softmax warp
    // keys that all of the warp's rows see, and that any does
    const int all_lo = __reduce_max_sync(0xffffffffu, vis.begin), all_hi = __reduce_min_sync(0xffffffffu, vis.end);
    const bool sees = vis.end > vis.begin;
    const int any_lo = __reduce_min_sync(0xffffffffu, sees ? vis.begin : INT_MAX);
    const int any_hi = __reduce_max_sync(0xffffffffu, sees ? vis.end : 0);
    const uint32_t s_addr = TM_S + mine * DQ_KEYS + lane_base + half * 32;
    const uint32_t dp_addr = TM_DP + mine * DQ_KEYS + lane_base + half * 32;
    const float ndl = s_row[r];
    const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
    const float C = ALIBI ? 1.f : p.c_log2;
    float rest = 0.f;  // sum of P (dP - delta) over this thread's keys
    for (int i = mine; i < n && ok; i += 2) {
      const int k0 = (kr.begin + i) * DQ_KEYS + half * 32, ph = (i >> 1) & 1;
      const bool padded = tile_has_pad(p, b, k0 / DA_TILE);
      if (!mbar_wait(&s_full[mine], ph, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      if (k0 >= any_hi || k0 + 32 <= any_lo) {  // nothing here is seen by the warp's rows
        if (!mbar_wait(&dp_full[mine], ph, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        uint32_t zero[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0u;
        tmem_st16(dp_addr, zero);
      } else {
      uint64_t x[16], f[CAP ? 16 : 1];  // scores, then P; the cap's derivative
      tmem_ld_pairs(s_addr, x);
      const bool masked = !(all_lo <= k0 && k0 + 32 <= all_hi);
      auto probabilities = [&](auto near) {
        const float fd = (float)(qpos - k0);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint64_t v = x[e];
          if (CAP) v = tanh2<decltype(near)::value, true>(v, p.x_scale, f[CAP ? e : 0]);
          if (ALIBI)
            v = fma2(f2(-slope2), f2(fabsf(fd - (float)(2 * e)), fabsf(fd - (float)(2 * e + 1))), mul2(v, f2(p.c_log2)));
          x[e] = ex2_2(fma2(v, f2(C), f2(nls)));
        }
      };
      if (CAP && warp_near(x, p.x_scale)) probabilities(std::true_type{});
      else probabilities(std::false_type{});
      if (!mbar_wait(&dp_full[mine], ph, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      // hidden pairs add nothing, whatever their scores and dP are
      auto gradients = [&](auto some_hidden) {
        constexpr bool HIDDEN = decltype(some_hidden)::value;
        const uint32_t bits = HIDDEN ? range_bits(vis.begin, vis.end, k0) : 0u;
        uint64_t rs = 0ull;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t d[16], pk[8];
          tmem_ld16(dp_addr + c * 16, d);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int t = c * 8 + e;
            uint64_t g = mul2(x[t], add2(f2(d[2 * e], d[2 * e + 1]), f2(ndl)));
            if (HIDDEN) g = select2(g, bits, 2 * t, 0.f);
            rs = add2(rs, g);
            if (CAP) g = mul2(g, f[CAP ? t : 0]);
            if (CAP && HIDDEN) g = select2(g, bits, 2 * t, 0.f);
            const float2 u = unpack2(g);
            pk[e] = pack_bf16(u.x, u.y);
          }
          tmem_st8(dp_addr + c * 8, pk);
        }
        const float2 rv = unpack2(rs);
        rest += rv.x + rv.y;
      };
      if (masked) gradients(std::true_type{});
      else gradients(std::false_type{});
      }
      // S_i has read K_i: rows of padding become zero before the dQ product reads them
      if (padded)
        zero_pad_rows<L::KBQ, DQ_KEYS>(sK + (i % L::ST) * L::K_BYTES, p, b, (kr.begin + i) * DQ_KEYS, half * 128 + r, 256);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[mine]);
    }
    if (ok && n > 0 && !mbar_wait(all_done, 0, abort_flag, p.status)) ok = false;
    s_row[(1 + sub) * DA_TILE + r] = rest;
    asm volatile("bar.sync 1, 512;" ::: "memory");  // reached by every softmax warp
    if (ok) {
      tc_fence_after();
      if (sub == 0 && in)
        ndelta[vi] = lone ? __uint_as_float(LONE_KEY)
                          : ndl - ((s_row[DA_TILE + r] + s_row[2 * DA_TILE + r]) +
                                   (s_row[3 * DA_TILE + r] + s_row[4 * DA_TILE + r]));
      // Q's tile in shared memory is free by now
      if (sub < L::KBQ)
        store_block(sQ, TM_DQ + lane_base, sub, p.Dqk, quarter, p.scale, n == 0, false, &tmDQ, h, qt * DA_TILE, p.S, b);
      if (lane == 0) bulk_wait_read<0>();
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
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const void* tmap, const void* smem_src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(tmap)),
               "r"(smem_u32(smem_src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// this thread's arrival, once its copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

constexpr int KV_QUERIES = 64;

template <int DQP, int DVP>
struct DaDkvSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int BLK = DA_TILE * 128, QBLK = KV_QUERIES * 128;
  static constexpr int K_BYTES = KBQ * BLK, V_BYTES = KBV * BLK, Q_BYTES = KBQ * QBLK, DO_BYTES = KBV * QBLK;
  static constexpr int ST = 4;  // Q / dO stages
  static constexpr int VEC = 4 * KV_QUERIES;  // -lse2, -delta, lo, hi of a step's queries
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + K_BYTES;
  static constexpr int OFF_Q = OFF_V + V_BYTES;
  static constexpr int OFF_DO = OFF_Q + ST * Q_BYTES;
  static constexpr int OFF_VEC = OFF_DO + ST * DO_BYTES;
  static constexpr int OFF_BAR = OFF_VEC + ST * VEC * 4;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

// Transposed tiles: TMEM lanes are keys, columns the 64 queries of a step.  TMEM: dV, dK, two buffers of S^T
// (then P^T) and of dP^T (then dS^T).  The softmax warps are two groups that take the steps in turn, each with
// its buffers: while a group works on its step the tensor cores work for the other's.  A warp owns 32 keys and
// 32 queries.
template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DA_GROUPS_THREADS, 1)
    da_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                  const __grid_constant__ CUtensorMap tmDK, const __grid_constant__ CUtensorMap tmDV, DaParams p,
                  const float* __restrict__ nlse2, const float* __restrict__ ndelta, int splits) {
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
  const int kt = blockIdx.z, hk = blockIdx.x / splits, part = blockIdx.x % splits, b = blockIdx.y;
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
    // K and V at once: the rest of the start runs under their latency
    mbar_arrive_expect_tx(kv_full, L::K_BYTES + L::V_BYTES);
#pragma unroll
    for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sK + kb * L::BLK, &tmK, kv_full, kb * 64, hk, kt * DA_TILE, b);
#pragma unroll
    for (int kb = 0; kb < L::KBV; ++kb) tma_load_4d(sV + kb * L::BLK, &tmV, kv_full, kb * 64, hk, kt * DA_TILE, b);
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmDO);
    tma_prefetch_desc(&tmDK);
    tma_prefetch_desc(&tmDV);
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
  const int first = (int)((int64_t)total * part / splits), n = (int)((int64_t)total * (part + 1) / splits) - first;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t TM_DV = tmem, TM_DK = tmem + 128, TM_S = tmem + 256, TM_DP = tmem + 384;

  if (warp == 0) {
    int it = 0;
    if (n > 0) {
      int h = hk * group + first / ni, qi = first % ni;
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
        // the step's vectors, asynchronously as well (waited for here, their latency set the steps' pace)
        const uint32_t vec = smem_u32(s_vec + st * L::VEC);
        const int64_t base = ((int64_t)b * p.Hq + h) * p.S;
#pragma unroll
        for (int c = 0; c < KV_QUERIES / 32; ++c) {
          const int q = c * 32 + lane, qpos = q0 + q;
          const bool in = qpos < p.S;  // past the end: zeros, and no key is seen
          const int64_t at = in ? qpos : 0;
          cp_async4(vec + q * 4, nlse2 + base + at, in);
          cp_async4(vec + (KV_QUERIES + q) * 4, ndelta + base + at, in);
          if (p.lo) {
            cp_async4(vec + (2 * KV_QUERIES + q) * 4, p.lo + (int64_t)b * p.S + at, in);
            cp_async4(vec + (3 * KV_QUERIES + q) * 4, p.hi + (int64_t)b * p.S + at, in);
          }
        }
        cp_async_arrive(&vec_full[st]);
        if (++qi == ni) {
          qi = 0;
          ++h;
        }
      }
    }
    if (lane == 0) {
      // leave no copy in flight into shared memory
      mbar_wait(kv_full, 0, nullptr, p.status);
      for (int u = max(0, it - L::ST); u < it; ++u) {
        mbar_wait(&q_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
        mbar_wait(&vec_full[u % L::ST], (u / L::ST) & 1, nullptr, p.status);
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
      bool hidden = false;  // none of the warp's queries sees any of its keys
      if (masked) {
        const int w0 = kt * DA_TILE + quarter * 32, q = q0 + half * 32 + lane;
        const int* range = reinterpret_cast<const int*>(s_vec + st * L::VEC + half * 32 + lane);
        const int lo = p.lo ? range[2 * KV_QUERIES] : 0;
        const int hi = p.lo ? range[3 * KV_QUERIES] : (q < p.S ? (p.causal ? q + 1 : p.S) : 0);
        hidden = !__any_sync(0xffffffffu, lo < w0 + 32 && hi > w0);
      }
      uint64_t x[16];  // scores, then P times the cap's derivative
      uint32_t pk[16];
      if (hidden) {
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = 0u;
      } else {
      tmem_ld_pairs(s_addr, x);
      auto probabilities = [&](auto near, auto some_hidden) {
        constexpr bool HIDDEN = decltype(some_hidden)::value;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 l4 = vec[e / 2];
          const uint64_t nls[2] = {f2(l4.x, l4.y), f2(l4.z, l4.w)};
          uint32_t sees = 15u;
          if (HIDDEN) {
            int lo[4] = {0, 0, 0, 0}, hi[4];
            if (p.lo) {
              const int4 a = ivec[2 * KV_QUERIES / 4 + e / 2], c = ivec[3 * KV_QUERIES / 4 + e / 2];
              lo[0] = a.x; lo[1] = a.y; lo[2] = a.z; lo[3] = a.w;
              hi[0] = c.x; hi[1] = c.y; hi[2] = c.z; hi[3] = c.w;
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int q = q0 + half * 32 + 2 * e + g;
                hi[g] = q < p.S ? (p.causal ? q + 1 : p.S) : 0;
              }
            }
            sees = 0u;
#pragma unroll
            for (int g = 0; g < 4; ++g) sees |= (lo[g] <= kpos && kpos < hi[g]) ? 1u << g : 0u;
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint64_t v = x[e + g], f = 0ull;
            if (CAP) v = tanh2<decltype(near)::value, true>(v, p.x_scale, f);
            if (ALIBI) {
              const float d = fd + (float)(2 * (e + g));
              v = fma2(f2(-slope2), f2(fabsf(d), fabsf(d + 1.f)), mul2(v, f2(p.c_log2)));
            }
            uint64_t pp = ex2_2(fma2(v, f2(C), nls[g]));
            if (HIDDEN) pp = select2(pp, sees, 2 * g, 0.f);
            if (CAP) {
              x[e + g] = mul2(pp, f);
              if (HIDDEN) x[e + g] = select2(x[e + g], sees, 2 * g, 0.f);  // a hidden pair's score may be NaN
            } else {
              x[e + g] = pp;
            }
            const float2 u = unpack2(pp);
            pk[e + g] = pack_bf16(u.x, u.y);
          }
        }
      };
      const bool near = CAP && warp_near(x, p.x_scale);
      if (masked) near ? probabilities(std::true_type{}, std::true_type{}) : probabilities(std::false_type{}, std::true_type{});
      else near ? probabilities(std::true_type{}, std::false_type{}) : probabilities(std::false_type{}, std::false_type{});
      }
      tmem_st16(s_addr, pk);
      if (padded) {
        // (dP^T may still be reading dO: only the columns of padded queries can differ, and those are not used)
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
      auto gradients = [&](auto some_hidden) {
        uint64_t d[16];
        tmem_ld_pairs(dp_addr, d);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 d4 = vec[KV_QUERIES / 4 + e / 2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float2 nd = g ? make_float2(d4.z, d4.w) : make_float2(d4.x, d4.y);
            const uint64_t ds = mul2(x[e + g], add2(d[e + g], f2(nd.x, nd.y)));
            float2 u = unpack2(ds);
            if (decltype(some_hidden)::value) {  // a hidden pair adds nothing, whatever dP is; nor does a lone key
              const float2 w = unpack2(x[e + g]);
              u.x = w.x == 0.f || __float_as_uint(nd.x) == LONE_KEY ? 0.f : u.x;
              u.y = w.y == 0.f || __float_as_uint(nd.y) == LONE_KEY ? 0.f : u.y;
            }
            pk[e + g] = pack_bf16(u.x, u.y);
          }
        }
      };
      if (hidden) {}  // pk is zero
      else if (masked) gradients(std::true_type{});
      else gradients(std::false_type{});
      tmem_st16(dp_addr, pk);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[mine]);
    }
    // K's and V's tiles are where the gradients are staged: without a step, their copies may still be on their way
    if (ok && !mbar_wait(n > 0 ? all_done : kv_full, 0, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
      // every product has completed and every copy landed: shared memory is free for the output tiles
      if (splits == 1) {
        for (int o = sub; o < L::KBV + L::KBQ; o += 4) {  // dV's, then dK's blocks of 64 columns
          if (o < L::KBV)
            store_block(sV, TM_DV + lane_base, o, p.Dv, quarter, 1.f, n == 0, false, &tmDV, hk, kt * DA_TILE, p.S, b);
          else
            store_block(sK, TM_DK + lane_base, o - L::KBV, p.Dqk, quarter, p.scale, n == 0, false, &tmDK, hk, kt * DA_TILE,
                        p.S, b);
        }
      } else {
        // f32 parts: 32 columns a store, staged in the Q / dO ring
        const int plane = (part * p.B + b) * p.Hk + hk;
        for (int o = sub; o < (DVP + DQP) / 32; o += 4) {
          const bool is_v = o < DVP / 32;
          const int c = is_v ? o : o - DVP / 32;
          uint8_t* slab = sQ + (o * 4 + quarter) * 4096;
          uint32_t w[32];
          tmem_ld32((is_v ? TM_DV : TM_DK) + lane_base + c * 32, w);
          tc_wait_ld();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = n == 0 ? 0u : __float_as_uint(__uint_as_float(w[q * 4 + e]) * (is_v ? 1.f : p.scale));
            sw128_store16(slab, lane, q, make_uint4(v[0], v[1], v[2], v[3]));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && c * 32 < (is_v ? p.Dv : p.Dqk) && kt * DA_TILE + quarter * 32 < p.S) {
            tma_store_3d(is_v ? &tmDV : &tmDK, slab, c * 32, kt * DA_TILE + quarter * 32, plane);
            bulk_commit();
          }
        }
      }
      if (lane == 0) bulk_wait_read<0>();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dV, dK = the splits' parts (f32 [split][B, Hk, S, D]) added in order; 8 columns a thread
__global__ void __launch_bounds__(256) da_join_kernel(const float* __restrict__ part_v, const float* __restrict__ part_k,
                                                      int splits, int B, int S, int Hk, int Dqk, int Dv,
                                                      __nv_bfloat16* __restrict__ dk, int64_t ldk,
                                                      __nv_bfloat16* __restrict__ dv, int64_t ldv) {
  const int vec = (Dqk + Dv) / 8;
  const int64_t rows = (int64_t)B * Hk * S, total = rows * vec;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int c0 = (int)(i % vec) * 8;
    const bool is_v = c0 < Dv;
    const int c = is_v ? c0 : c0 - Dv, D = is_v ? Dv : Dqk;
    const int64_t row = i / vec, s = row % S, bh = row / S, h = bh % Hk, b = bh / Hk;
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < splits; ++q) {
      const float4* src = reinterpret_cast<const float4*>((is_v ? part_v : part_k) + (q * rows + row) * D + c);
      const float4 x = __ldg(src), y = __ldg(src + 1);
      a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w;
      a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
    }
    __nv_bfloat16* dst = is_v ? dv + (b * S + s) * ldv + h * Dv + c : dk + (b * S + s) * ldk + h * Dqk + c;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(a[4], a[5]),
                                                pack_bf16(a[6], a[7]));
  }
}

// f32 [planes, S, D]: boxes of 32 columns x 32 rows
inline CUtensorMap part_tmap(float* ptr, int64_t planes, int S, int D) {
  ensure_current_context();
  CUtensorMap m;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)D * 4, (cuuint64_t)S * D * 4};
  cuuint32_t box[3] = {32, 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = get_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, ptr, dims, strides, box, estr,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  OXI_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (gradient parts) failed: ", (int)r);
  return m;
}

struct BwdArgs {
  DaShape s;
  DaTensor q, k, v, o, o_lo, dout;
  const float* nlse2;
  float *ndelta, *part;
  DaOut dq, dk, dv;
  int* status;
  cudaStream_t st;
};

template <int DQP, int DVP, bool CAP, bool ALIBI>
void launch_bwd_t(const BwdArgs& a) {
  const DaShape& s = a.s;
  const DaParams p = da_params(s, a.status);
  const CUtensorMap tq = da_tmap(a.q, s.B, s.S, s.Hq, s.Dqk), td = da_tmap(a.dout, s.B, s.S, s.Hq, s.Dv),
                    tk = da_tmap(a.k, s.B, s.S, s.Hk, s.Dqk), tv = da_tmap(a.v, s.B, s.S, s.Hk, s.Dv),
                    tk64 = da_tmap(a.k, s.B, s.S, s.Hk, s.Dqk, DQ_KEYS), tv64 = da_tmap(a.v, s.B, s.S, s.Hk, s.Dv, DQ_KEYS),
                    tq64 = da_tmap(a.q, s.B, s.S, s.Hq, s.Dqk, KV_QUERIES),
                    td64 = da_tmap(a.dout, s.B, s.S, s.Hq, s.Dv, KV_QUERIES),
                    tdq = da_tmap_out(a.dq, s.B, s.S, s.Hq, s.Dqk);
  auto kq = da_dq_kernel<DQP, DVP, CAP, ALIBI>;
  auto kkv = da_dkv_kernel<DQP, DVP, CAP, ALIBI>;
  static std::atomic<uint64_t> dq_devices{0}, dkv_devices{0};
  set_smem_once(kq, DaDqSmem<DQP, DVP>::TOTAL, dq_devices);
  set_smem_once(kkv, DaDkvSmem<DQP, DVP>::TOTAL, dkv_devices);
  kq<<<dim3(s.Hq, s.B, p.nt), DA_GROUPS_THREADS, DaDqSmem<DQP, DVP>::TOTAL, a.st>>>(tq, tk64, tv64, td, tdq, p, a.o, a.o_lo,
                                                                                    a.nlse2, a.ndelta);
  OXI_CUDA_CHECK(cudaGetLastError());
  const int splits = da_bwd_splits(s.B, s.S, s.Hq, s.Hk);
  const int64_t planes = (int64_t)splits * s.B * s.Hk;
  float* part_k = a.part ? a.part + planes * s.S * s.Dv : nullptr;
  const CUtensorMap tdk = splits > 1 ? part_tmap(part_k, planes, s.S, s.Dqk) : da_tmap_out(a.dk, s.B, s.S, s.Hk, s.Dqk),
                    tdv = splits > 1 ? part_tmap(a.part, planes, s.S, s.Dv) : da_tmap_out(a.dv, s.B, s.S, s.Hk, s.Dv);
  kkv<<<dim3(s.Hk * splits, s.B, p.nt), DA_GROUPS_THREADS, DaDkvSmem<DQP, DVP>::TOTAL, a.st>>>(
      tq64, tk, tv, td64, tdk, tdv, p, a.nlse2, a.ndelta, splits);
  OXI_CUDA_CHECK(cudaGetLastError());
  if (splits > 1) {
    const int64_t threads = (int64_t)s.B * s.Hk * s.S * ((s.Dqk + s.Dv) / 8);
    da_join_kernel<<<(unsigned)std::min<int64_t>((threads + 255) / 256, 148 * 16), 256, 0, a.st>>>(
        a.part, part_k, splits, s.B, s.S, s.Hk, s.Dqk, s.Dv, reinterpret_cast<__nv_bfloat16*>(a.dk.ptr), a.dk.ld,
        reinterpret_cast<__nv_bfloat16*>(a.dv.ptr), a.dv.ld);
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
                   const DaTensor& o_lo, const DaTensor& dout, const float* nlse2, float* ndelta, float* part,
                   const DaOut& dq, const DaOut& dk, const DaOut& dv, int* status, cudaStream_t st) {
  if (s.B == 0 || s.S == 0 || s.Hq == 0) return;
  da_check(s);
  for (const DaOut* t : {&dq, &dk, &dv})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->ld % 8 == 0, "16-byte aligned gradient rows");
  for (const DaTensor* t : {&o, &o_lo, &dout})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->sb % 8 == 0 && t->ss % 8 == 0 && t->sh % 8 == 0,
              "16-byte aligned rows of the output and its gradient");
  OXI_CHECK(da_bwd_splits(s.B, s.S, s.Hq, s.Hk) == 1 || part != nullptr, "attention backward needs its parts' workspace");
  const BwdArgs a{s, q, k, v, o, o_lo, dout, nlse2, ndelta, part, dq, dk, dv, status, st};
  if (s.Dqk <= 64 && s.Dv <= 64) launch_bwd_d<64, 64>(a);
  else if (s.Dv <= 64) launch_bwd_d<128, 64>(a);
  else launch_bwd_d<128, 128>(a);
}

}  // namespace oxi
