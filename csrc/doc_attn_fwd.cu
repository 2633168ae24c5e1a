// Attention over visible key ranges for sm_100a (tcgen05 + TMEM + TMA), forward.
//
//   z_ij = scale q_i . k_j,  u = cap tanh(z / cap) (or z),  a = u - slope_h |i - j|
//   o_i  = sum_{lo_i <= j < hi_i} softmax(a_i)_j v_j      (a row that sees nothing: 0)
//
// One CTA per (128 queries, query head, batch), two CTAs on an SM: while one is between its tiles, or
// at its start or end (documents are short, so that is often), the other works.  Q stays in shared
// memory; K/V tiles of 64 keys stream through TMA rings.  Per step of 64 keys:
//   S  = Q K^T              tcgen05.mma into one of two TMEM buffers, a step ahead
//   P  = 2^(S - m)          one thread per query row, its 64 keys in registers, no exchange between
//                           threads; P (bf16) goes back over S in TMEM
//   O += P V                tcgen05.mma with A = P from TMEM
// The reference m need not be the row's maximum, it has only to keep 2^(S - m) in range: a step takes
// the m of the steps before it, so that its exponentials wait for no maximum, and the maximum found
// meanwhile moves m (and rescales O in TMEM) for the next step when it is more than 8 above.  Only
// where it is more than 60 above, or a row sees its first keys, is the step's own maximum used.
// O is divided by the sum of the rounded P: it is then a true mean of the v_j, with weights a rounding off,
// and where one key has nearly all the weight its rounding cancels.  The backward's delta lives on that (see
// doc_attn_bwd.cu); its P takes the sum of P itself.  For a backward, what rounding o to bf16 leaves over is
// kept as a second bf16 (o_lo).  (Both together: 166 -> 185 us in the capped case below.  The second sum is taken
// without a backward too, so that o is the same.)
// Scores capped at up to 60 log 2 need no maximum at all: m = 0 (unless a negative slope adds to them).
// Steps outside the bounds of the query tile's ranges are not loaded or computed; a step that is
// wholly visible to a warp's 32 rows is computed without a mask.
// Warps: 0 TMA, 1 MMA + TMEM owner, 2..5 softmax and output.
//
// What bounds it: a step's products take 652 clocks (128-wide heads), its 8192 exponentials 512 of the
// special-function unit, and neither runs alone: 1100 clocks a step.  One dense causal row of 8192 tokens, 16 / 4
// heads: 261 us of width 128 (1054 TFLOP/s), 239 us of width 64 (575; the exponentials alone take 120 us at
// the unit's rate), 406 us of width 128 under a cap of 50.  8 x 2048 tokens in documents of 700 with that cap: 185 us;
// 16 x 1024 in documents of 300, 96- and 64-wide heads: 58 us, of which a CTA's six steps are the smaller part
// (start, first loads and output take 4 us, which the other CTA of the SM covers only while it computes).
// Tried and slower: eight softmax warps that halve a row (they exchange maxima and sums at each step).
#include "doc_attn.cuh"

namespace oxi {
namespace {

constexpr int FW_KEYS = 64;
constexpr int FW_THREADS = 192;

template <int DQP, int DVP>
struct DaFwdSmem {
  static constexpr int KBQ = DQP / 64, KBV = DVP / 64;
  static constexpr int QBLK = DA_TILE * 128, KBLK = FW_KEYS * 128;  // blocks of 64 columns
  static constexpr int Q_BYTES = KBQ * QBLK, K_BYTES = KBQ * KBLK, V_BYTES = KBV * KBLK;
  static constexpr int KST = 2, VST = 2;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + Q_BYTES;
  static constexpr int OFF_V = OFF_K + KST * K_BYTES;
  static constexpr int OFF_BAR = OFF_V + VST * V_BYTES;
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(2 * (TOTAL + 1024) <= 233472, "two CTAs per SM");
};

template <int DQP, int DVP, bool CAP, bool ALIBI>
__global__ void __launch_bounds__(FW_THREADS, 2)
    da_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                  const __grid_constant__ CUtensorMap tmOlo, DaParams p, float* __restrict__ nlse2, bool want_lo) {
  using L = DaFwdSmem<DQP, DVP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + L::OFF_Q;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;   // [2]
  uint64_t* k_empty = bars + 3;  // [2]
  uint64_t* v_full = bars + 5;   // [2]
  uint64_t* v_empty = bars + 7;  // [2]
  uint64_t* s_full = bars + 9;   // [2] per S buffer
  uint64_t* p_full = bars + 11;  // [2]
  uint64_t* pv_done = bars + 13;
  uint64_t* o_done = bars + 14;  // the last product
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  // the query tile is the slowest grid index and runs backwards: the longest causal rows start first
  const int qt = gridDim.z - 1 - blockIdx.z, h = blockIdx.x, b = blockIdx.y;
  const int hk = h / (p.Hq / p.Hk);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(o_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    // Q at once: the rest of the start runs under its latency
    mbar_arrive_expect_tx(q_full, L::Q_BYTES);
#pragma unroll
    for (int kb = 0; kb < L::KBQ; ++kb) tma_load_4d(sQ + kb * L::QBLK, &tmQ, q_full, kb * 64, h, qt * DA_TILE, b);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmO);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  const TileRange kr = key_steps(p, b, qt, FW_KEYS);
  const int n = kr.end - kr.begin;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t TM_S = tmem, TM_O = tmem + 2 * FW_KEYS;

  if (warp == 0) {
    if (lane == 0) {
      int ki = 0, vi = 0;
      for (; ki < n; ++ki) {
        const int st = ki % L::KST;
        if (!mbar_wait(&k_empty[st], ((ki / L::KST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(&k_full[st], L::K_BYTES);
#pragma unroll
        for (int kb = 0; kb < L::KBQ; ++kb)
          tma_load_4d(sK + st * L::K_BYTES + kb * L::KBLK, &tmK, &k_full[st], kb * 64, hk, (kr.begin + ki) * FW_KEYS, b);
        // V_j is asked for once K_{j+1} has been: K is needed a step earlier
        bool ok = true;
        for (; ok && vi < n && (vi < ki || ki == n - 1); ++vi) {
          const int sv = vi % L::VST;
          ok = mbar_wait(&v_empty[sv], ((vi / L::VST) & 1) ^ 1, abort_flag, p.status);
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[sv], L::V_BYTES);
#pragma unroll
          for (int kb = 0; kb < L::KBV; ++kb)
            tma_load_4d(sV + sv * L::V_BYTES + kb * L::KBLK, &tmV, &v_full[sv], kb * 64, hk, (kr.begin + vi) * FW_KEYS, b);
        }
        if (!ok) { ++ki; break; }
      }
      // leave no copy in flight into shared memory
      mbar_wait(q_full, 0, nullptr, p.status);
      for (int i = max(0, ki - L::KST); i < ki; ++i) mbar_wait(&k_full[i % L::KST], (i / L::KST) & 1, nullptr, p.status);
      for (int i = max(0, vi - L::VST); i < vi; ++i) mbar_wait(&v_full[i % L::VST], (i / L::VST) & 1, nullptr, p.status);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (n > 0) {
      const uint32_t lead = elect_lead();
      constexpr uint32_t ID_S = umma_idesc_bf16(DA_TILE, FW_KEYS, false, false);
      constexpr uint32_t ID_O = umma_idesc_bf16(DA_TILE, DVP, false, true);
      const int nkk = (p.Dqk + 15) / 16;
      const DaDesc dQ = da_desc(smem_u32(sQ), 16);
      bool ok = warp_wait(q_full, 0, abort_flag, p.status);
      // S_i's buffer last held P_{i-2}, read by a product issued before
      auto issue_s = [&](int i) -> bool {
        if (!warp_wait(&k_full[i % L::KST], (i / L::KST) & 1, abort_flag, p.status)) return false;
        tc_fence_after();
        da_mma_kk<DQP, L::QBLK, L::KBLK>(lead, TM_S + (i & 1) * FW_KEYS, dQ,
                                         da_desc(smem_u32(sK + (i % L::KST) * L::K_BYTES), 16), ID_S, nkk);
        da_commit(lead, &s_full[i & 1]);
        da_commit(lead, &k_empty[i % L::KST]);
        return true;
      };
      if (ok) ok = issue_s(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n && !issue_s(i + 1)) { ok = false; break; }
        if (!warp_wait(&v_full[i % L::VST], (i / L::VST) & 1, abort_flag, p.status) ||
            !warp_wait(&p_full[i & 1], (i >> 1) & 1, abort_flag, p.status)) { ok = false; break; }
        tc_fence_after();
        const DaDesc dV = da_desc(smem_u32(sV + (i % L::VST) * L::V_BYTES), L::KBLK);
#pragma unroll
        for (int kk = 0; kk < FW_KEYS / 16; ++kk)
          da_mma_ts(lead, TM_O, TM_S + (i & 1) * FW_KEYS + kk * 8, dV.at(kk * 2048), ID_O,
                        (i | kk) != 0);
        da_commit(lead, pv_done);
        da_commit(lead, &v_empty[i % L::VST]);
        if (i + 1 == n) da_commit(lead, o_done);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;  // TMEM lanes a warp may read: 32 * (warp % 4)
    const int r = quarter * 32 + lane;
    const int qpos = qt * DA_TILE + r;
    const TileRange vis = key_range(p, b, qpos);
    // keys that all rows of the warp see
    const int all_lo = __reduce_max_sync(0xffffffffu, vis.begin), all_hi = __reduce_min_sync(0xffffffffu, vis.end);
    // keys that any of them sees
    const bool sees = vis.end > vis.begin;
    const int any_lo = __reduce_min_sync(0xffffffffu, sees ? vis.begin : INT_MAX);
    const int any_hi = __reduce_max_sync(0xffffffffu, sees ? vis.end : 0);
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const float slope2 = ALIBI ? __ldg(p.slopes + h) * LOG2E : 0.f;
    const float C = ALIBI ? 1.f : p.c_log2;
    const bool bounded = CAP && p.c_log2 <= 60.f && slope2 >= 0.f;
    float m = bounded ? 0.f : -INFINITY, m_next = m, l = 0.f, lr = 0.f;  // sums of P and of the rounded P
    bool ok = true;
    // O times 2^(m - m_new), m = m_new; O belongs to the product of step i - 1 until it completes.  Called
    // behind S_i, which was issued after the product of step i - 2: pv_done's parity can only mean i - 1.
    auto move = [&](int i, float m_new) -> bool {
      const float alpha = m_new == m ? 1.f : ex2_approx(m - m_new);  // 2^-inf = 0 at a row's first keys
      m = m_new;
      l *= alpha;
      lr *= alpha;
      if (i == 0) return true;
      if (!mbar_wait(pv_done, (i - 1) & 1, abort_flag, p.status)) return false;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < DVP / 32; ++c) {
        uint32_t w[32];
        tmem_ld32(TM_O + lane_base + c * 32, w);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * alpha);
        tmem_st32(TM_O + lane_base + c * 32, w);
      }
      tc_wait_st();
      return true;
    };
    for (int i = 0; i < n; ++i) {
      const int k0 = (kr.begin + i) * FW_KEYS;
      const bool padded = tile_has_pad(p, b, k0 / DA_TILE);
      const uint32_t s_addr = TM_S + (i & 1) * FW_KEYS + lane_base;
      if (!mbar_wait(&s_full[i & 1], (i >> 1) & 1, abort_flag, p.status)) { ok = false; break; }
      tc_fence_after();
      if (!bounded && __any_sync(0xffffffffu, m_next > m) && !move(i, m_next)) { ok = false; break; }
      if (k0 >= any_hi || k0 + FW_KEYS <= any_lo) {  // nothing here is seen by the warp's rows
        uint32_t zero[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) zero[e] = 0u;
        tmem_st32(s_addr, zero);
      } else {
      uint64_t x[2][16];
      {
        uint32_t w[2][32];
        tmem_ld32(s_addr, w[0]);
        tmem_ld32(s_addr + 32, w[1]);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e >> 4][e & 15] = f2(w[e >> 4][2 * (e & 15)], w[e >> 4][2 * (e & 15) + 1]);
      }
      const bool masked = !(all_lo <= k0 && k0 + FW_KEYS <= all_hi);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (CAP) {
          uint64_t unused;
          auto capped = [&](auto near) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[c][e] = tanh2<decltype(near)::value, false>(x[c][e], p.x_scale, unused);
          };
          if (warp_near(x[c], p.x_scale)) capped(std::true_type{});
          else capped(std::false_type{});
        }
        if (ALIBI) {
          const float fd = (float)(qpos - (k0 + c * 32));
#pragma unroll
          for (int e = 0; e < 16; ++e)
            x[c][e] = fma2(f2(-slope2), f2(fabsf(fd - (float)(2 * e)), fabsf(fd - (float)(2 * e + 1))),
                           mul2(x[c][e], f2(p.c_log2)));
        }
        if (masked) {
          const uint32_t bits = range_bits(vis.begin, vis.end, k0 + c * 32);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[c][e] = select2(x[c][e], bits, 2 * e, -INFINITY);
        }
      }
      uint32_t pk[2][16];
      uint64_t rs[4];
      auto exponentials = [&]() {
        const uint64_t mref = f2(m == -INFINITY ? 0.f : -m), cc = f2(C);
#pragma unroll
        for (int q = 0; q < 4; ++q) rs[q] = 0ull;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t pp = ex2_2(fma2(x[c][e], cc, mref));
            const float2 v = unpack2(pp);
            pk[c][e] = pack_bf16(v.x, v.y);
            rs[e & 1] = add2(rs[e & 1], pp);
            rs[2 + (e & 1)] = add2(rs[2 + (e & 1)], f2(pk[c][e] << 16, pk[c][e] & 0xffff0000u));
          }
      };
      exponentials();
      if (!bounded) {
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 v = unpack2(x[e >> 4][e & 15]);
          mx[e & 3] = fmaxf(fmaxf(v.x, v.y), mx[e & 3]);
        }
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * C;
        if (__any_sync(0xffffffffu, m == -INFINITY ? mt > -INFINITY : mt > m + 60.f)) {
          if (!move(i, fmaxf(mt, m))) { ok = false; break; }
          exponentials();
        }
        m_next = mt > m + 8.f ? mt : m;
      }
      tmem_st16(s_addr, pk[0]);
      tmem_st16(s_addr + 16, pk[1]);
      const float2 exact = unpack2(add2(rs[0], rs[1])), rounded = unpack2(add2(rs[2], rs[3]));
      l += exact.x + exact.y;
      lr += rounded.x + rounded.y;
      }
      if (padded) {
        // V_i has landed before its product may read it; rows of padding become zero
        if (!mbar_wait(&v_full[i % L::VST], (i / L::VST) & 1, abort_flag, p.status)) { ok = false; break; }
        zero_pad_rows<L::KBV, FW_KEYS>(sV + (i % L::VST) * L::V_BYTES, p, b, k0, r, 128);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i & 1]);
    }
    // Q's tile is where the output is staged: without a step, its copy may still be on its way
    if (ok && !mbar_wait(n > 0 ? o_done : q_full, 0, abort_flag, p.status)) ok = false;
    if (ok) {
      tc_fence_after();
      // a row that sees no key is zero; one whose scores are NaN stays NaN.  the tiles in shared memory are free
      const bool some = lr > 0.f;
      const float inv = some ? 1.f / lr : 0.f;
      static_assert(L::KBV * L::QBLK <= L::KST * L::K_BYTES, "o_lo is staged in K's ring");
#pragma unroll 1
      for (int kb = 0; kb < L::KBV; ++kb) {
        if (want_lo)
          store_block<true>(sQ, TM_O + lane_base, kb, p.Dv, quarter, inv, !some, l != l, &tmO, h, qt * DA_TILE, p.S, b, sK,
                            &tmOlo);
        else
          store_block(sQ, TM_O + lane_base, kb, p.Dv, quarter, inv, !some, l != l, &tmO, h, qt * DA_TILE, p.S, b);
      }
      if (qpos < p.S) nlse2[((int64_t)b * p.Hq + h) * p.S + qpos] = l == 0.f ? -INFINITY : -(m + log2f(l));
      if (lane == 0) bulk_wait_read<0>();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <int DQP, int DVP, bool CAP, bool ALIBI>
void launch_fwd_t(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                  const DaOut& o_lo, float* nlse2, int* status, cudaStream_t st) {
  using L = DaFwdSmem<DQP, DVP>;
  const CUtensorMap tq = da_tmap(q, s.B, s.S, s.Hq, s.Dqk), tk = da_tmap(k, s.B, s.S, s.Hk, s.Dqk, FW_KEYS),
                    tv = da_tmap(v, s.B, s.S, s.Hk, s.Dv, FW_KEYS), to = da_tmap_out(o, s.B, s.S, s.Hq, s.Dv),
                    tlo = o_lo.ptr ? da_tmap_out(o_lo, s.B, s.S, s.Hq, s.Dv) : to;
  auto kern = da_fwd_kernel<DQP, DVP, CAP, ALIBI>;
  static std::atomic<uint64_t> devices{0};
  set_smem_once(kern, L::TOTAL, devices);
  const dim3 grid(s.Hq, s.B, (s.S + DA_TILE - 1) / DA_TILE);
  kern<<<grid, FW_THREADS, L::TOTAL, st>>>(tq, tk, tv, to, tlo, da_params(s, status), nlse2, o_lo.ptr != nullptr);
  OXI_CUDA_CHECK(cudaGetLastError());
}

template <int DQP, int DVP>
void launch_fwd_d(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                  const DaOut& o_lo, float* nlse2, int* status, cudaStream_t st) {
  if (s.cap > 0.f)
    s.slopes ? launch_fwd_t<DQP, DVP, true, true>(s, q, k, v, o, o_lo, nlse2, status, st)
             : launch_fwd_t<DQP, DVP, true, false>(s, q, k, v, o, o_lo, nlse2, status, st);
  else
    s.slopes ? launch_fwd_t<DQP, DVP, false, true>(s, q, k, v, o, o_lo, nlse2, status, st)
             : launch_fwd_t<DQP, DVP, false, false>(s, q, k, v, o, o_lo, nlse2, status, st);
}

}  // namespace

bool da_supported(int Dqk, int Dv) {
  return Dqk >= 8 && Dv >= 8 && Dqk <= 128 && Dv <= 128 && Dqk % 8 == 0 && Dv % 8 == 0;
}

void launch_da_fwd(const DaShape& s, const DaTensor& q, const DaTensor& k, const DaTensor& v, const DaOut& o,
                   const DaOut& o_lo, float* nlse2, int* status, cudaStream_t st) {
  if (s.B == 0 || s.S == 0 || s.Hq == 0) return;
  da_check(s);
  for (const DaOut* t : {&o, &o_lo})
    OXI_CHECK((reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->ld % 8 == 0, "16-byte aligned output rows");
  // kernels for widths of up to 64 and 128 columns: narrower heads are padded with zero columns
  if (s.Dqk <= 64 && s.Dv <= 64) launch_fwd_d<64, 64>(s, q, k, v, o, o_lo, nlse2, status, st);
  else if (s.Dv <= 64) launch_fwd_d<128, 64>(s, q, k, v, o, o_lo, nlse2, status, st);
  else launch_fwd_d<128, 128>(s, q, k, v, o, o_lo, nlse2, status, st);
}

}  // namespace oxi
