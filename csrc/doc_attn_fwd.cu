// Attention over visible key ranges for sm_100a (tcgen05 + TMEM + TMA), forward.
//
//   z_ij = scale q_i . k_j,  u = cap tanh(z / cap) (or z),  a = u - slope_h |i - j|
//   o_i  = sum_{lo_i <= j < hi_i} softmax(a_i)_j v_j      (a row that sees nothing: 0)
//
// One CTA per (256 queries, query head, batch): two query tiles of 128 that take turns, so that
// one tile's softmax runs while the tensor cores work for the other.  K/V tiles of 128 keys stream
// through a TMA ring and serve both.  Per tile and key tile:
//   S  = Q K^T              tcgen05.mma into TMEM
//   P  = 2^(S - m)          one thread per query row, 128 keys in registers, no exchange between
//                           threads; P (bf16) goes back over S in TMEM
//   O += P V                tcgen05.mma with A = P from TMEM
// The running maximum m moves (and O is rescaled in TMEM) only when it grows by more than 2^8.
// Key tiles outside the bounds of a query tile's ranges are not loaded or computed; a tile that
// is wholly visible to a warp's 32 rows is computed without a mask.
// Warps: 0 TMA, 1 MMA + TMEM owner, 2..5 softmax of query tile 0, 6..9 of query tile 1.
#include "doc_attn.cuh"

namespace oxi {
namespace {

template <int DQP, int DVP>
struct DaFwdSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int BLK = DA_TILE * 128;  // 128 rows x 64 columns
  static constexpr int Q_BYTES = KBQ * BLK, V_BYTES = KBV * BLK;
  static constexpr int KST = 2, VST = 2;
  static constexpr int OFF_Q = 0;                          // [2] query tiles
  static constexpr int OFF_K = OFF_Q + 2 * Q_BYTES;
  static constexpr int OFF_V = OFF_K + KST * Q_BYTES;
  static constexpr int OFF_BAR = OFF_V + VST * V_BYTES;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(TOTAL <= 232448, "shared memory budget");
};

template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(DA_THREADS, 1)
    da_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, DaParams p, __nv_bfloat16* __restrict__ o_out, int64_t ldo,
                  float* __restrict__ lse2) {
  using L = DaFwdSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + L::OFF_Q;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;    // [2]
  uint64_t* k_empty = bars + 3;   // [2]
  uint64_t* v_full = bars + 5;    // [2]
  uint64_t* v_empty = bars + 7;   // [2]
  uint64_t* s_full = bars + 9;    // [2] per query tile
  uint64_t* p_full = bars + 11;   // [2]
  uint64_t* pv_done = bars + 13;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // the query tile is the slowest grid index and runs backwards: the longest causal rows start first
  const int pair = gridDim.z - 1 - blockIdx.z;
  const int h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (p.Hq / p.Hk);
  const TileRange r0 = key_tiles(p, b, 2 * pair), r1 = key_tiles(p, b, 2 * pair + 1);
  const bool a0 = r0.end > r0.begin, a1 = r1.end > r1.begin;
  const int j_begin = a0 && a1 ? min(r0.begin, r1.begin) : (a0 ? r0.begin : r1.begin);
  const int j_end = a0 && a1 ? max(r0.end, r1.end) : (a0 ? r0.end : r1.end);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto tm_s = [&](int t) { return tmem + t * DA_TILE; };
  auto tm_o = [&](int t) { return tmem + 2 * DA_TILE + t * DVP; };
  const int n = j_end - j_begin;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(q_full, 2 * L::Q_BYTES);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sQ + t * L::Q_BYTES + kb * L::BLK, &tmQ, q_full, kb * 64, h, (2 * pair + t) * DA_TILE, b);
      int ki = 0, vi = 0;
      for (; ki < n; ++ki) {
        const int st = ki % L::KST;
        if (!mbar_wait(&k_empty[st], ((ki / L::KST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(&k_full[st], L::Q_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sK + st * L::Q_BYTES + kb * L::BLK, &tmK, &k_full[st], kb * 64, hk, (j_begin + ki) * DA_TILE, b);
        const int sv = vi % L::VST;
        if (!mbar_wait(&v_empty[sv], ((vi / L::VST) & 1) ^ 1, abort_flag, p.status)) { ++ki; break; }
        mbar_arrive_expect_tx(&v_full[sv], L::V_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBV; ++kb)
          tma_load_4d(sV + sv * L::V_BYTES + kb * L::BLK, &tmV, &v_full[sv], kb * 64, hk, (j_begin + vi) * DA_TILE, b);
        ++vi;
      }
      // leave no copy in flight into shared memory
      mbar_wait(q_full, 0, nullptr, p.status);
      for (int i = max(0, ki - L::KST); i < ki; ++i) mbar_wait(&k_full[i % L::KST], (i / L::KST) & 1, nullptr, p.status);
      for (int i = max(0, vi - L::VST); i < vi; ++i) mbar_wait(&v_full[i % L::VST], (i / L::VST) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, DA_TILE, false, false);
      constexpr uint32_t ID_O = umma_idesc_bf16(DA_TILE, DVP, false, true);
      const int nkk = (p.Dqk + 15) / 16;
      const TileRange rt[2] = {r0, r1};
      int done[2] = {0, 0};  // PV products issued per query tile
      bool ok = mbar_wait(q_full, 0, abort_flag, p.status);
      auto active = [&](int t, int j) { return j >= rt[t].begin && j < rt[t].end; };
      // S of query tile t and key tile j_begin + i (in stage i % KST, already waited for); its
      // buffer last held P of the previous key tile, read by the PV product issued before
      auto issue_s = [&](int t, int i) {
        const uint32_t aQ = smem_u32(sQ + t * L::Q_BYTES), aK = smem_u32(sK + (i % L::KST) * L::Q_BYTES);
        for (int kk = 0; kk < nkk; ++kk)
          tc_mma_f16(tm_s(t), da_kmajor_desc(aQ, kk, L::BLK), da_kmajor_desc(aK, kk, L::BLK), ID_S, kk != 0);
        tc_commit(&s_full[t]);
      };
      auto wait_k = [&](int i) {
        return mbar_wait(&k_full[i % L::KST], (i / L::KST) & 1, abort_flag, p.status);
      };
      if (ok) ok = wait_k(0);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (active(t, j_begin)) issue_s(t, 0);
        tc_commit(&k_empty[0]);
      }
      for (int i = 0; i < n && ok; ++i) {
        const int j = j_begin + i;
        if (i + 1 < n && !wait_k(i + 1)) { ok = false; break; }
        if (!mbar_wait(&v_full[i % L::VST], (i / L::VST) & 1, abort_flag, p.status)) { ok = false; break; }
        const uint32_t aV = smem_u32(sV + (i % L::VST) * L::V_BYTES);
        for (int t = 0; t < 2 && ok; ++t) {
          if (active(t, j)) {
            if (!mbar_wait(&p_full[t], done[t] & 1, abort_flag, p.status)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < DA_TILE / 16; ++kk)
              tc_mma_f16_ts(tm_o(t), tm_s(t) + kk * 8, umma_desc_sw128(aV + kk * 2048, L::BLK, 1024), ID_O,
                            (done[t] | kk) != 0);
            tc_commit(&pv_done[t]);
            ++done[t];
          }
          if (i + 1 < n && active(t, j + 1)) {
            tc_fence_after();
            issue_s(t, i + 1);
          }
        }
        tc_commit(&v_empty[i % L::VST]);
        if (i + 1 < n) tc_commit(&k_empty[(i + 1) % L::KST]);
      }
    }
    __syncwarp();
  } else {
    const int t = (warp - 2) >> 2;  // query tile of this warp
    const int quarter = warp & 3;   // TMEM lanes a warp may read: 32 * (warp % 4)
    const int r = quarter * 32 + lane;
    const TileRange rt = t == 0 ? r0 : r1;
    const int qpos = (2 * pair + t) * DA_TILE + r;
    const TileRange vis = key_range(p, b, qpos);
    // keys that all / any rows of the warp see
    const int all_lo = __reduce_max_sync(0xffffffffu, vis.begin), all_hi = __reduce_min_sync(0xffffffffu, vis.end);
    const uint32_t s_addr = tm_s(t) + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_addr = tm_o(t) + ((uint32_t)(quarter * 32) << 16);
    const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
    const float C = ALIBI ? 1.f : p.c_log2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const int nj = rt.end - rt.begin;
    for (int i = 0; i < nj; ++i) {
      const int j = rt.begin + i, k0 = j * DA_TILE;
      if (!mbar_wait(&s_full[t], i & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, x[c]);
      tc_wait_ld();
      const bool masked = !(all_lo <= k0 && k0 + DA_TILE <= all_hi);
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (CAP || ALIBI) {
          const float fd = (float)(qpos - (k0 + c * 32));
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float v = __uint_as_float(x[c][e]);
            if (CAP) v = tanh_ex2(v * p.x_scale);
            if (ALIBI) v = fmaf(-slope2, fabsf(fd - (float)e), v * p.c_log2);
            x[c][e] = __float_as_uint(v);
          }
        }
        if (masked) {
          const uint32_t bits = range_bits(vis.begin, vis.end, k0 + c * 32);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((bits >> e) & 1u)) x[c][e] = 0xff800000u;  // -inf
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(x[c][e]));
      }
      const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * C;
      const bool move = mt > m + 8.f;
      const float m_new = move ? mt : m;
      const float alpha = move ? ex2_approx(m - m_new) : 1.f;  // 2^-inf = 0 at a row's first keys
      const float mref = m_new == -INFINITY ? 0.f : m_new;
      m = m_new;
      if (i > 0 && __any_sync(0xffffffffu, move)) {
        // O belongs to the previous product until it completes
        if (!mbar_wait(&pv_done[t], (i - 1) & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DVP / 32; ++c) {
          uint32_t w[32];
          tmem_ld32(o_addr + c * 32, w);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * alpha);
          tmem_st32(o_addr + c * 32, w);
        }
        tc_wait_st();
      }
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float a = ex2_approx(fmaf(__uint_as_float(x[c][e]), C, -mref));
          const float bb = ex2_approx(fmaf(__uint_as_float(x[c][e + 1]), C, -mref));
          rs[(e >> 1) & 3] += a + bb;
          pk[e / 2] = pack_bf16(a, bb);
        }
        tmem_st16(s_addr + c * 16, pk);
      }
      l = l * alpha + ((rs[0] + rs[1]) + (rs[2] + rs[3]));
      if (tile_has_pad(p, b, j)) {
        // V_j has landed before its product may read it; rows of padding become zero
        if (!mbar_wait(&v_full[(j - j_begin) % L::VST], ((j - j_begin) / L::VST) & 1, abort_flag, p.status)) {
          ok = false;
          break;
        }
        zero_pad_rows<L::KBV>(sV + ((j - j_begin) % L::VST) * L::V_BYTES, p, b, k0, r, 128);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && nj > 0 && !mbar_wait(&pv_done[t], (nj - 1) & 1, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
      const bool valid = qpos < p.S;
      const float inv_l = l > 0.f ? 1.f / l : 0.f;
      __nv_bfloat16* orow = o_out + ((int64_t)b * p.S + qpos) * ldo + (int64_t)h * p.Dv;
#pragma unroll 1
      for (int c = 0; c < DVP / 32; ++c) {
        uint32_t w[32];
        if (nj > 0) {
          tmem_ld32(o_addr + c * 32, w);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) w[e] = 0u;
        }
        if (valid) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (c * 32 + q * 8 < p.Dv) {
              uint32_t u[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                u[e] = l > 0.f ? pack_bf16(__uint_as_float(w[q * 8 + 2 * e]) * inv_l,
                                           __uint_as_float(w[q * 8 + 2 * e + 1]) * inv_l)
                               : (l == l ? 0u : 0x7fff7fffu);  // no visible key: 0; NaN scores stay NaN
              *reinterpret_cast<uint4*>(orow + c * 32 + q * 8) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
        }
      }
      if (valid) lse2[((int64_t)b * p.Hq + h) * p.S + qpos] = l == 0.f ? INFINITY : m + log2f(l);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DQP, int DVP, bool CAP, bool ALIBI>
void launch_fwd_t(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                  float* lse2, int* status, cudaStream_t st) {
  using L = DaFwdSmem<DQP, DVP>;
  const CUtensorMap tq = da_tmap(q, s.B, s.S, s.Hq, s.Dqk), tk = da_tmap(k, s.B, s.S, s.Hk, s.Dqk),
                    tv = da_tmap(v, s.B, s.S, s.Hk, s.Dv);
  auto kern = da_fwd_kernel<DQP, DVP, CAP, ALIBI>;
  da_smem(kern, L::TOTAL);
  const dim3 grid(s.Hq, s.B, (s.S + 2 * DA_TILE - 1) / (2 * DA_TILE));
  kern<<<grid, DA_THREADS, L::TOTAL, st>>>(tq, tk, tv, da_params(s, status), reinterpret_cast<__nv_bfloat16*>(o.ptr),
                                           o.ld, lse2);
  OXI_CUDA_CHECK(cudaGetLastError());
}

template <int DQP, int DVP>
void launch_fwd_d(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                  float* lse2, int* status, cudaStream_t st) {
  if (s.cap > 0.f)
    s.slopes ? launch_fwd_t<DQP, DVP, true, true>(s, q, k, v, o, lse2, status, st)
             : launch_fwd_t<DQP, DVP, true, false>(s, q, k, v, o, lse2, status, st);
  else
    s.slopes ? launch_fwd_t<DQP, DVP, false, true>(s, q, k, v, o, lse2, status, st)
             : launch_fwd_t<DQP, DVP, false, false>(s, q, k, v, o, lse2, status, st);
}

}  // namespace

bool da_supported(int Dqk, int Dv) {
  return Dqk >= 8 && Dv >= 8 && Dqk <= 128 && Dv <= 128 && Dqk % 8 == 0 && Dv % 8 == 0;
}

void launch_da_fwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                   float* lse2, int* status, cudaStream_t st) {
  if (s.B == 0 || s.S == 0 || s.Hq == 0) return;
  da_check(s);
  OXI_CHECK((reinterpret_cast<uintptr_t>(o.ptr) & 15) == 0 && o.ld % 8 == 0, "16-byte aligned output rows");
  // kernels for widths of up to 64 and 128 columns: narrower heads are padded with zero columns
  if (s.Dqk <= 64 && s.Dv <= 64) launch_fwd_d<64, 64>(s, q, k, v, o, lse2, status, st);
  else if (s.Dv <= 64) launch_fwd_d<128, 64>(s, q, k, v, o, lse2, status, st);
  else launch_fwd_d<128, 128>(s, q, k, v, o, lse2, status, st);
}

}  // namespace oxi
