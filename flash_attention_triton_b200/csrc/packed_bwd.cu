// Causal attention backward over packed sequences with grouped heads (packed.cuh).
//
// The arithmetic, the warp roles and the tensor-memory plans are those of dkdv_roles (mode 0, bwd_roles.cuh) and
// bwd_dq_kernel (bwd.cu).  A CTA of the dK / dV kernel has one KV tile of a key head and walks the Q tiles of ALL query heads
// that share it, one head after the other, so dK and dV are summed over them in tensor memory, in a fixed order and
// without another pass; a CTA of the dQ kernel has one Q tile of a query head.  Both recompute the scores, so
// no memory beyond O(rows) is needed and the same call gives the same bits.  P and dS enter the second products in 16 bits, the
// type that the tensor pipe takes beside dO, Q and K: the gradients' error against exact ones is 1.4 to 1.5 times that of their own
// rounding, up to 1.65 times on sequences of few rows, where delta has the rounding of O.
// Bound by the tensor pipe: seven products where five would do.  bf16, 23 202 rows in three sequences, 16 / 4 heads of
// 128 columns, each kernel alone: dK / dV 1 118 us (four products, 1 474 GFLOP, tensor pipe 74 % active), dQ 913 us (three products, 64 %);
// in a loop under the power limit 1 245 and 1 112.  Handing dS over through memory would save two of the seven products; it
// takes scratch that is quadratic in the lengths, 8.6 GB for all 16 heads at once and 2.1 for four at a time, and a caller who says the longest.
#include "bwd_roles.cuh"
#include "packed.cuh"

namespace fa2 {
namespace {

// 32 rows of a warp from a [128, KD] fp32 accumulator as 16 bits, times `mul`: through a free tile buffer and the tensor map
// where all 32 belong to the sequence (`left` >= 32), row by row where only the first `left` do.  `parts` of the same rows
// from other CTAs, `part_stride` floats apart, are added first: [KD / 4][32 lanes][4] floats each.
template <int D, bool BF16, int KD>
__device__ __forceinline__ void store_packed_rows(uint32_t tmem_row_addr, uint8_t* stage, int warp4, int lane,
                                                  const CUtensorMap* map, int row, int head, int heads, int left, void* out,
                                                  int cols, float mul, const float* part = nullptr, int parts = 0,
                                                  int part_stride = 0) {
  using T = Tile<D>;
  const bool whole = left >= 32;
  uint16_t* const dst = static_cast<uint16_t*>(out) + (static_cast<long long>(row + lane) * heads + head) * cols;
#pragma unroll
  for (int c0 = 0; c0 < KD; c0 += 32) {
    uint32_t v[32];
    tmem_ld_x32(tmem_row_addr + c0, v);
    tmem_wait_ld();
    float* const f = reinterpret_cast<float*>(v);
    for (int i = 0; i < parts; ++i)
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float4 x = reinterpret_cast<const float4*>(part + i * part_stride)[(c0 / 4 + p) * 32 + lane];
        f[4 * p] += x.x, f[4 * p + 1] += x.y, f[4 * p + 2] += x.z, f[4 * p + 3] += x.w;
      }
    const int piece0 = (c0 % T::kChunkElems) / 8;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint4 val;
      val.x = pack2<BF16>(f[8 * p + 0] * mul, f[8 * p + 1] * mul);
      val.y = pack2<BF16>(f[8 * p + 2] * mul, f[8 * p + 3] * mul);
      val.z = pack2<BF16>(f[8 * p + 4] * mul, f[8 * p + 5] * mul);
      val.w = pack2<BF16>(f[8 * p + 6] * mul, f[8 * p + 7] * mul);
      if (whole)
        *reinterpret_cast<uint4*>(stage + c0 / T::kChunkElems * T::kChunkTileBytes + swizzled_offset<D>(warp4 * 32 + lane, piece0 + p)) = val;
      else if (lane < left && c0 + 8 * p < cols)
        *reinterpret_cast<uint4*>(dst + c0 + 8 * p) = val;
    }
  }
  if (!whole) return;
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    for (int ch = 0; ch < (KD + T::kChunkElems - 1) / T::kChunkElems; ++ch)
      tma_store_4d(map, ch * T::kChunkElems, row, HeadCoord{head, 0}, smem_u32(stage + ch * T::kChunkTileBytes + warp4 * 32 * T::kRowBytes));
    tma_store_commit();
    tma_store_wait_all();
  }
}

// The power of two that dS carries at fp16 (head_dscale), by the largest |dO| of `heads` query heads from `head` on.  For dQ that is
// the one head of the product; for dK and dV all of a key head, because their products meet in one accumulator.  bf16 has the
// exponents of fp32 and needs none.
template <bool BF16>
__device__ __forceinline__ float heads_dscale(const PackedStats& stats, int capacity, int base, int tiles, int head, int heads,
                                              int lane, float* inverse) {
  if constexpr (BF16) {
    *inverse = 1.f;
    return 1.f;
  } else {
    const int words = 4 * tiles;  // of a head, one behind the other
    unsigned m = 0;
    for (int i = lane; i < heads * words; i += 32) {
      const int h = i / words;
      m = max(m, ld_global(stats.amax + (static_cast<size_t>(head + h) * capacity + base) * 4 + (i - h * words)));
    }
    return dscale_of<false>(__reduce_max_sync(0xffffffffu, m), inverse);
  }
}

// =========================================================================================
// dK / dV: one CTA per KV tile of a key head, or a cluster of two or four (S) that share its query heads
// =========================================================================================
// A KV tile with G query heads is G times the work of one, and there are G times fewer of them, so with few tiles a launch
// waits for the longest of them.  The CTAs of a cluster then share the query heads, and the 128 rows.  At their end each sends
// its fp32 accumulators of the rows that another one owns into that one's idle rings: no memory, no
// other launch, one order of the sum.  When: packed_cluster.
template <int D, bool BF16, int KD, int W, int S>
__global__ void __launch_bounds__(DkdvCfg<D, 0, W>::kThreads, DkdvCfg<D, 0, W>::kCtasPerSm)
    packed_dkdv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                       const __grid_constant__ CUtensorMap tdk, const __grid_constant__ CUtensorMap tdv, void* dk, void* dv,
                       const PackedTile* list, const int* counts, PackedStats stats, int capacity, int Hkv, int G, int cols,
                       float scale, float scale_log2, int* status) {
  using C = DkdvCfg<D, 0, W>;
  using T = Tile<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = ((threadIdx.x >> 5) + C::kMmaWarp) % (C::kThreads / 32), lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  if (smem_base & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, 0x20000 | kBSiteAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_base + C::kOffBar + 8u * i; };
  if (threadIdx.x == 0) {
    dkdv_init_barriers<D, 0, W>(smem_base + C::kOffBar);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const WaitCtx w{abort_flag, status};
  grid_wait_previous();
  if (blockIdx.x == 0 && threadIdx.x == 0) release_flag(stats.written);
  grid_allow_next();

  static_assert(S == 1 || S == 2 || S == 4, "packed_cluster");
  const int rank = S == 1 ? 0 : blockIdx.x % S, entry = blockIdx.x / S / Hkv, kv_head = blockIdx.x / S - entry * Hkv;
  const int first_head = kv_head * G + rank * (G / S);  // of this CTA's query heads
  if (entry < ld_global(counts)) {
  const PackedTile e = load_tile(list + entry);
  const int ntiles = (e.length + 127) >> 7;
  const int nq = e.tile + 1, jt = ntiles - nq;  // Q tiles ntiles - 1 down to jt meet KV tile jt
  const int row_k = e.row0 + jt * 128, left = e.length - jt * 128;  // rows of the KV tile in the sequence
  // A Q tile is worked through in kSub steps of W rows, first rows first (dkdv_roles).
  constexpr int kSub = 128 / W;
  const int per_head = nq * kSub, nsteps = per_head * (G / S);
  const HeadCoord hk{kv_head, 0};
  // step u of a query head: first row in the sequence
  auto q_row = [&](int u) { return (ntiles - 1 - u / kSub) * 128 + (u % kSub) * W; };

  if (warp >= C::kMmaWarp) {
    reg_dec<C::kProducerRegs>();
    if (warp == C::kLoadWarp) {
      const uint32_t elected = elect_one();
      if (elected) {
        prefetch_tensormap(&tq);
        prefetch_tensormap(&tdo);
        mbar_arrive_expect_tx(bar(C::kBarKV), 2 * T::kTileBytes);
        for (int ch = 0; ch < T::kChunks; ++ch) {
          tma_load_4d(smem_base + C::kOffK + ch * T::kChunkTileBytes, &tk, ch * T::kChunkElems, row_k, hk, bar(C::kBarKV));
          tma_load_4d(smem_base + C::kOffV + ch * T::kChunkTileBytes, &tv, ch * T::kChunkElems, row_k, hk, bar(C::kBarKV));
        }
      }
      int s = 0, ph = 1;
      bool ok = true;
      for (int g = 0; ok && g < G / S; ++g) {
        const HeadCoord hq{first_head + g, 0};
        const float* head_stats = stats.stats + (static_cast<size_t>(hq.h) * capacity + e.base) * 256;
        for (int u = 0; u < per_head; ++u) {
          const int row = q_row(u);
          if (!(ok = mbar_wait_warp(bar(C::kBarQEmpty + s), ph, w, kBSiteLoadQ))) break;
          if (elected) {
            mbar_arrive_expect_tx(bar(C::kBarQFull + s), C::kStepBytes + W * 8);
#pragma unroll
            for (int ch = 0; ch < T::kChunks; ++ch)
              tma_load_4d(smem_base + C::kOffQ + s * C::kStepBytes + ch * (C::kStepBytes / T::kChunks), &tq, ch * T::kChunkElems,
                          e.row0 + row, hq, bar(C::kBarQFull + s));
            const float* from = head_stats + static_cast<size_t>(row >> 7) * 256 + (row & 127);
            bulk_load_1d(smem_base + C::kOffStats + s * W * 8, from, W * 4, bar(C::kBarQFull + s));
            bulk_load_1d(smem_base + C::kOffStats + s * W * 8 + W * 4, from + 128, W * 4, bar(C::kBarQFull + s));
          }
          if (!(ok = mbar_wait_warp(bar(C::kBarDOEmpty + s), ph, w, kBSiteLoadDO))) break;
          if (elected) {
            mbar_arrive_expect_tx(bar(C::kBarDOFull + s), C::kStepBytes);
#pragma unroll
            for (int ch = 0; ch < T::kChunks; ++ch)
              tma_load_4d(smem_base + C::kOffDO + s * C::kStepBytes + ch * (C::kStepBytes / T::kChunks), &tdo, ch * T::kChunkElems,
                          e.row0 + row, hq, bar(C::kBarDOFull + s));
          }
          if (++s == C::kStages) s = 0, ph ^= 1;
        }
      }
    } else if (warp == C::kMmaWarp || warp == C::kMmaWarp + 2) {
      // The two MMA-issuing warps X and Y of dkdv_roles.  Their waits vote, because clear_rows wants a converged warp.
      const uint32_t elected = elect_one();
      const uint32_t ka = smem_base + C::kOffK, va = smem_base + C::kOffV;
      auto commit = [&](int b) {
        if (elected) mma_commit(bar(b));
      };
      bool ok = mbar_wait_warp(bar(C::kBarKV), 0, w, kBSiteMmaKV);
      int s = 0, ph = 0;  // ring stage / phase of step t
      int u1 = 0;         // step t + 1 within its query head
      constexpr uint32_t kHalf = C::kCols;
      auto next_u = [&](int u) { return u + 1 == per_head ? 0 : u + 1; };
      if (warp == C::kMmaWarp) {
        // ------------------------------------------------------------ warp X: St(t + 1) = K Q^T, dV += Pt dO
        auto score = [&](int stage, int u) {
          clear_rows<D, W>(smem + C::kOffQ + stage * C::kStepBytes, e.length - q_row(u), lane);
          issue_rows_x_rows<D, BF16, W, KD>(elected, tmem_base + C::kColSt, ka, smem_base + C::kOffQ + stage * C::kStepBytes);
        };
        if (ok && (ok = mbar_wait_warp(bar(C::kBarQFull + 0), 0, w, kBSiteMmaQ))) {
          score(0, 0);
          commit(C::kBarStFull + 0);
          commit(C::kBarQEmpty + 0);
        }
        for (int t = 0, u = 0; ok && t < nsteps; ++t, u = u1) {
          u1 = next_u(u);
          const int s1 = s + 1 == C::kStages ? 0 : s + 1, ph1 = s1 ? ph : ph ^ 1;  // of step t+1
          if (!(ok = mbar_wait_warp(bar(C::kBarDOFull + s), ph, w, kBSiteMmaDO))) break;
          if (!(ok = mbar_wait_warp(bar(C::kBarPtReady), t & 1, w, kBSiteMmaPt))) break;
          tc_fence_after();
          clear_rows<D, W>(smem + C::kOffDO + s * C::kStepBytes, e.length - q_row(u), lane);
          issue_tmem_x_tile<D, BF16, W, KD>(elected, tmem_base + C::kColDV, tmem_base + C::kColSt, kHalf,
                                        smem_base + C::kOffDO + s * C::kStepBytes, t > 0);
          commit(C::kBarDOEmpty + s);
          if (t + 1 < nsteps) {
            if (!(ok = mbar_wait_warp(bar(C::kBarQFull + s1), ph1, w, kBSiteMmaQ))) break;
            score(s1, u1);
            commit(C::kBarStFull + (t + 1) % C::kStBars);
            commit(C::kBarQEmpty + s1);
          }
          s = s1;
          ph = ph1;
        }
        if (ok) commit(C::kBarDone);
      } else {
        // ------------------------------------------------------------ warp Y: dPt(t + 1) = V dO^T, dK += dSt Q
        auto products = [&](int stage, int u) {
          clear_rows<D, W>(smem + C::kOffDO + stage * C::kStepBytes, e.length - q_row(u), lane);
          issue_rows_x_rows<D, BF16, W, KD>(elected, tmem_base + C::kColDpt, va, smem_base + C::kOffDO + stage * C::kStepBytes);
        };
        if (ok && (ok = mbar_wait_warp(bar(C::kBarDOFull + 0), 0, w, kBSiteMmaDO))) {
          products(0, 0);
          commit(C::kBarDptFull);
          commit(C::kBarDOEmpty + 0);
        }
        for (int t = 0, u = 0; ok && t < nsteps; ++t, u = u1) {
          u1 = next_u(u);
          const int s1 = s + 1 == C::kStages ? 0 : s + 1, ph1 = s1 ? ph : ph ^ 1;
          if (!(ok = mbar_wait_warp(bar(C::kBarQFull + s), ph, w, kBSiteMmaQ))) break;
          if (!(ok = mbar_wait_warp(bar(C::kBarDsReady), t & 1, w, kBSiteMmaDs))) break;
          // St(t+1) sits on the critical chain St -> Pt -> dV -> St: warp X gets it into the pipe first
          if (t + 1 < nsteps &&
              !(ok = mbar_wait_warp(bar(C::kBarStFull + (t + 1) % C::kStBars), ((t + 1) / C::kStBars) & 1, w, kBSiteMmaQ)))
            break;
          tc_fence_after();
          // Q of step t is as warp X has cleared it: dSt needed St
          issue_tmem_x_tile<D, BF16, W, KD>(elected, tmem_base + C::kColDK, tmem_base + C::kColDpt, kHalf,
                                        smem_base + C::kOffQ + s * C::kStepBytes, t > 0);
          commit(C::kBarQEmpty + s);
          if (t + 1 < nsteps) {
            if (!(ok = mbar_wait_warp(bar(C::kBarDOFull + s1), ph1, w, kBSiteMmaDO))) break;
            products(s1, u1);
            commit(C::kBarDptFull);
            commit(C::kBarDOEmpty + s1);
          }
          s = s1;
          ph = ph1;
        }
        if (ok) commit(C::kBarDone);
      }
    }
    __syncwarp();
    if constexpr (S > 1) {
      cluster_sync();
      cluster_sync();
    }
  } else {
    // ---------------------------------------------------------------- compute groups
    reg_inc<C::kComputeRegs>();
    constexpr int kCols = C::kCols, kPairs = kCols / 2;
    const int wg = warp >> 2;  // score columns (q) wg * kCols ..
    const int w4 = warp & 3;
    const int r = w4 * 32 + lane;  // kv row in the tile = tensor-memory lane
    const uint32_t lane_base = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t tSt = tmem_base + lane_base + C::kColSt + wg * kCols;
    const uint32_t tDpt = tmem_base + lane_base + C::kColDpt + wg * kCols;
    const float2 sc2 = make_float2(scale_log2, scale_log2);
    float inv_dscale;
    const float dscale = heads_dscale<BF16>(stats, capacity, e.base, ntiles, kv_head * G, G, lane, &inv_dscale);
    const float ds_scale = scale * dscale * kProbabilityInverse<BF16>;  // dS = P (dP - delta) scale 2^k
    const float2 scale2 = make_float2(ds_scale, ds_scale);
    bool ok = true;
    for (int t = 0, u = 0; t < nsteps; ++t, u = u + 1 == per_head ? 0 : u + 1) {
      const int s = t % C::kStages, ph = (t / C::kStages) & 1;
      const int row = q_row(u), qt = row >> 7;
      const float* st = reinterpret_cast<const float*>(smem + C::kOffStats + s * (W * 8));
      const float4* nlse = reinterpret_cast<const float4*>(st + wg * kCols);      // -lse*log2e (+ kProbabilityPower)
      const float4* ndlt = reinterpret_cast<const float4*>(st + W + wg * kCols);  // -delta
      if (!(ok = mbar_wait_warp(bar(C::kBarQFull + s), ph, w, kBSiteCmpQ))) break;
      if (!(ok = mbar_wait_warp(bar(C::kBarStFull + t % C::kStBars), (t / C::kStBars) & 1, w, kBSiteCmpSt))) break;
      tc_fence_after();
      float2 p[kPairs];  // P^T for this thread's kv row, q columns wg*kCols ..
      {
        uint32_t sr[kCols];
#pragma unroll
        for (int c = 0; c < kCols; c += 32) tmem_ld_x32(tSt + c, sr + c);
        tmem_wait_ld();
        probabilities_of_row<kPolyShareT<D>>(sr, nlse, sc2, p);
      }
      // diagonal tile: keep q >= kv; rows behind the sequence keep nothing (their dK and dV are not stored)
      if (qt == jt || left < 128) mask_row(p, r >= left ? 128 : (qt == jt ? r : 0), (row & 127) + wg * kCols);
      {
        uint32_t pk[kPairs];
#pragma unroll
        for (int c = 0; c < kPairs; ++c) pk[c] = pack2<kInterBF16<BF16>>(p[c].x, p[c].y);
        if constexpr (kPairs == 16) tmem_st_x16(tSt, pk); else tmem_st_x32(tSt, pk);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kBarPtReady));

      if (!(ok = mbar_wait_warp(bar(C::kBarDptFull), t & 1, w, kBSiteCmpDpt))) break;
      tc_fence_after();
      uint32_t dsk[kPairs];
#pragma unroll
      for (int h = 0; h < kCols / 32; ++h) {
        uint32_t dp[32];
        tmem_ld_x32(tDpt + 32 * h, dp);
        tmem_wait_ld();
#pragma unroll
        for (int c4 = 0; c4 < 8; ++c4) {
          const float4 nd = ndlt[8 * h + c4];
          float2 u0 = __fadd2_rn(make_float2(__uint_as_float(dp[4 * c4]), __uint_as_float(dp[4 * c4 + 1])), make_float2(nd.x, nd.y));
          float2 u1 = __fadd2_rn(make_float2(__uint_as_float(dp[4 * c4 + 2]), __uint_as_float(dp[4 * c4 + 3])), make_float2(nd.z, nd.w));
          u0 = __fmul2_rn(__fmul2_rn(p[16 * h + 2 * c4], u0), scale2);
          u1 = __fmul2_rn(__fmul2_rn(p[16 * h + 2 * c4 + 1], u1), scale2);
          dsk[16 * h + 2 * c4] = pack2<kInterBF16<BF16>>(u0.x, u0.y);
          dsk[16 * h + 2 * c4 + 1] = pack2<kInterBF16<BF16>>(u1.x, u1.y);
        }
      }
      if constexpr (kPairs == 16) tmem_st_x16(tDpt, dsk); else tmem_st_x32(tDpt, dsk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kBarDsReady));
    }
    // epilogue: group 0 has dV, group 1 dK; staged through the idle V and K tiles
    ok = ok && mbar_wait_warp(bar(C::kBarDone), 0, w, kBSiteCmpDone);
    tc_fence_after();
    const uint32_t sums = tmem_base + lane_base + (wg == 0 ? C::kColDV : C::kColDK);
    constexpr int kWarpsOfRank = 4 / S, kPartFloats = KD * 32;  // warps of a group whose rows a CTA owns; floats of 32 rows
    const int owner = w4 / kWarpsOfRank;
    // parts that arrive here: [sender, without the receiver][dV, dK][warp of the owner][KD / 4][32 lanes][4]
    const int at = (wg * kWarpsOfRank + w4 % kWarpsOfRank) * kPartFloats;
    constexpr int kSenderFloats = 2 * kWarpsOfRank * kPartFloats;
    static_assert(S == 1 || (S - 1) * kSenderFloats * 4 <= 2 * C::kStages * C::kStepBytes, "the rings take the parts");
    if constexpr (S > 1) {
      cluster_sync();  // every CTA has formed its last product: the rings are idle
      if (ok && owner != rank) {
        const uint32_t to = cluster_address(smem_base + C::kOffQ + ((rank < owner ? rank : rank - 1) * kSenderFloats + at) * 4, owner);
#pragma unroll
        for (int c0 = 0; c0 < KD; c0 += 32) {
          uint32_t v[32];
          tmem_ld_x32(sums + c0, v);
          tmem_wait_ld();
#pragma unroll
          for (int p = 0; p < 8; ++p) st_cluster_v4(to + ((c0 / 4 + p) * 32 + lane) * 16, v + 4 * p);
        }
      }
      cluster_sync();
    }
    if (ok && owner == rank)
      store_packed_rows<D, BF16, KD>(sums, smem + (wg == 0 ? C::kOffV : C::kOffK), w4, lane, wg == 0 ? &tdv : &tdk, row_k + w4 * 32,
                                     kv_head, Hkv, left - w4 * 32, wg == 0 ? dv : dk, cols, wg == 0 ? kProbabilityInverse<BF16> : inv_dscale,
                                     reinterpret_cast<const float*>(smem + C::kOffQ) + at, S - 1, kSenderFloats);
  }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// =========================================================================================
// dQ: one CTA per Q tile of a query head, KV tiles in ascending order
// =========================================================================================
// It needs nothing of the dK / dV kernel in front of it, which reads no output, so its CTAs work as soon as they find room, under
// that one's last CTAs (a kernel for both needs one CTA to an SM for dQ as well: 99.2).  fp16, eight sequences of 256 to 1024 rows, 16 / 4 heads of 64 columns, whole training pass: 101.6 us when they wait, 89.1;
// 4096 rows, backward alone 163 and 155.
template <int D, int W>
struct PackedDqCfg {
  using T = Tile<D>;
  static_assert(W == 128 || (W == 64 && D <= 64), "packed_step_rows");
  static constexpr int kCtasPerSm = W == 64 ? 2 : 1;
  static constexpr int kCols = W / 2;  // score columns of a compute thread
  static constexpr int kKvBytes = T::kTileBytes / 128 * W;
  static constexpr int kKStages = W == 64 ? 4 : 3;  // K_j is needed by S(j) and, later, by dQ(j)
  static constexpr int kVStages = W == 64 ? 3 : 2;
  static constexpr int kMmaWarp = 8;
  static constexpr int kThreads = 384;
  static constexpr int kLoadWarp = kMmaWarp + 1;
  static constexpr int kLaunchRegs = 65536 / (kThreads * kCtasPerSm) / 8 * 8;
  static constexpr int kProducerRegs = W == 64 ? 48 : 72;
  static constexpr int kComputeRegs = W == 64 ? 96 : 208;
  static_assert(128 * kProducerRegs + 256 * kComputeRegs <= kThreads * kLaunchRegs,
                "setmaxnreg.inc waits for registers that setmaxnreg.dec has released");
  static constexpr int kOffQ = 0;
  static constexpr int kOffDO = kOffQ + T::kTileBytes;
  static constexpr int kOffK = kOffDO + T::kTileBytes;
  static constexpr int kOffV = kOffK + kKStages * kKvBytes;
  static constexpr int kOffStats = kOffV + kVStages * kKvBytes;  // [256] fp32
  static constexpr int kOffBar = kOffStats + 1024;
  static constexpr int kBarQ = 0;  // Q, dO and row statistics
  static constexpr int kBarKFull = 1;
  static constexpr int kBarKEmpty = kBarKFull + kKStages;
  static constexpr int kBarVFull = kBarKEmpty + kKStages;
  static constexpr int kBarVEmpty = kBarVFull + kVStages;
  static constexpr int kBarSFull = kBarVEmpty + kVStages;  // 2 (one per score buffer)
  static constexpr int kBarDpFull = kBarSFull + 2;
  static constexpr int kBarDpConsumed = kBarDpFull + 1;  // one arrival per compute warp
  static constexpr int kBarDsReady = kBarDpConsumed + 1;  // 2, by j % 2 (DqCfg in bwd.cu)
  static constexpr int kBarDqDone = kBarDsReady + 2;      // 2: dQ += dS(j) K_j completed, by j % 2
  static constexpr int kBarDone = kBarDqDone + 2;
  static constexpr int kNumBars = kBarDone + 1;
  static constexpr int kSmemBytes = kOffBar + kNumBars * 8 + 16;
  static constexpr int kColS = 0;  // score buffers at 0 and W; dS (16-bit) overwrites them
  static constexpr int kColDp = 2 * W;
  static constexpr int kColDQ = 3 * W;
  static constexpr int kTmemCols = 512 / kCtasPerSm;
  static_assert(kColDQ + D <= kTmemCols, "tensor memory of one CTA");
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory of one SM");
};

template <int D, bool BF16, int KD, int W>
__global__ void __launch_bounds__(PackedDqCfg<D, W>::kThreads, PackedDqCfg<D, W>::kCtasPerSm)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                     const __grid_constant__ CUtensorMap tdq, void* dq, const PackedTile* list, const int* counts,
                     PackedStats stats, int capacity, int Hq, int G, int cols, float scale, float scale_log2, int* status) {
  using C = PackedDqCfg<D, W>;
  using T = Tile<D>;
  constexpr int kCols = C::kCols, kPairs = kCols / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = ((threadIdx.x >> 5) + C::kMmaWarp) % (C::kThreads / 32), lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  if (smem_base & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, 0, 0x20000 | kBSiteAlign);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_base + C::kOffBar + 8u * i; };

  if (threadIdx.x == 0) {
    mbar_init(bar(C::kBarQ), 1);
    for (int i = 0; i < C::kKStages; ++i) {
      mbar_init(bar(C::kBarKFull + i), 1);
      mbar_init(bar(C::kBarKEmpty + i), 2);  // S(j) and dQ(j) both done
    }
    for (int i = 0; i < C::kVStages; ++i) {
      mbar_init(bar(C::kBarVFull + i), 1);
      mbar_init(bar(C::kBarVEmpty + i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(C::kBarSFull + i), 1);
      mbar_init(bar(C::kBarDsReady + i), 8);
      mbar_init(bar(C::kBarDqDone + i), 1);
    }
    mbar_init(bar(C::kBarDpFull), 1);
    mbar_init(bar(C::kBarDpConsumed), 8);
    mbar_init(bar(C::kBarDone), 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const WaitCtx w{abort_flag, status};
  grid_wait_unless(stats.written);
  grid_allow_next();

  const int entry = blockIdx.x / Hq, head = blockIdx.x - entry * Hq;
  if (entry < ld_global(counts)) {
  const PackedTile e = load_tile(list + entry);
  const int qt = e.tile, row_q = e.row0 + qt * 128;
  const HeadCoord hq{head, 0}, hk{head / G, 0};
  // steps of W keys up to the diagonal, or to the last key
  const int nkv = min((qt + 1) * (128 / W), (e.length + W - 1) / W);
  auto commit_to = [&](uint32_t elected, int b) {
    if (elected) mma_commit(bar(b));
  };

  if (warp >= C::kMmaWarp) {
    reg_dec<C::kProducerRegs>();
    if (warp == C::kLoadWarp) {
      const uint32_t elected = elect_one();
      if (elected) {
        prefetch_tensormap(&tk);
        prefetch_tensormap(&tv);
        mbar_arrive_expect_tx(bar(C::kBarQ), 2 * T::kTileBytes + 1024);
        for (int ch = 0; ch < T::kChunks; ++ch) {
          tma_load_4d(smem_base + C::kOffQ + ch * T::kChunkTileBytes, &tq, ch * T::kChunkElems, row_q, hq, bar(C::kBarQ));
          tma_load_4d(smem_base + C::kOffDO + ch * T::kChunkTileBytes, &tdo, ch * T::kChunkElems, row_q, hq, bar(C::kBarQ));
        }
        bulk_load_1d(smem_base + C::kOffStats, stats.stats + (static_cast<size_t>(head) * capacity + e.base + qt) * 256, 1024, bar(C::kBarQ));
      }
      for (int j = 0; j < nkv; ++j) {
        const int ks = j % C::kKStages, kph = (j / C::kKStages) & 1;
        if (!mbar_wait_warp(bar(C::kBarKEmpty + ks), kph ^ 1, w, kBSiteLoadQ)) break;
        if (elected) {
          mbar_arrive_expect_tx(bar(C::kBarKFull + ks), C::kKvBytes);
#pragma unroll
          for (int ch = 0; ch < T::kChunks; ++ch)
            tma_load_4d(smem_base + C::kOffK + ks * C::kKvBytes + ch * (C::kKvBytes / T::kChunks), &tk, ch * T::kChunkElems,
                        e.row0 + j * W, hk, bar(C::kBarKFull + ks));
        }
        const int vs = j % C::kVStages, vph = (j / C::kVStages) & 1;
        if (!mbar_wait_warp(bar(C::kBarVEmpty + vs), vph ^ 1, w, kBSiteLoadDO)) break;
        if (elected) {
          mbar_arrive_expect_tx(bar(C::kBarVFull + vs), C::kKvBytes);
#pragma unroll
          for (int ch = 0; ch < T::kChunks; ++ch)
            tma_load_4d(smem_base + C::kOffV + vs * C::kKvBytes + ch * (C::kKvBytes / T::kChunks), &tv, ch * T::kChunkElems,
                        e.row0 + j * W, hk, bar(C::kBarVFull + vs));
        }
      }
    } else if (warp == C::kMmaWarp) {
      // ------------------------------------------------------------ warp X: dP(j) = dO V_j^T
      const uint32_t elected = elect_one();
      int vs = 0, vph = 0;  // ring position of the next V tile
      bool ok = mbar_wait_warp(bar(C::kBarQ), 0, w, kBSiteMmaQ);
      for (int j = 0; ok && j < nkv; ++j) {
        if (j > 0) {
          // dP columns are free once every compute warp has read dP(j-1)
          if (!(ok = mbar_wait_warp(bar(C::kBarDpConsumed), (j - 1) & 1, w, kBSiteMmaDrain))) break;
          tc_fence_after();
        }
        if (!(ok = mbar_wait_warp(bar(C::kBarVFull + vs), vph, w, kBSiteMmaDO))) break;
        // dS = P o (dP - delta) takes dP of a masked key times zero
        clear_rows<D, W>(smem + C::kOffV + vs * C::kKvBytes, e.length - j * W, lane);
        issue_rows_x_rows<D, BF16, W, KD>(elected, tmem_base + C::kColDp, smem_base + C::kOffDO,
                                   smem_base + C::kOffV + vs * C::kKvBytes);
        commit_to(elected, C::kBarDpFull);
        commit_to(elected, C::kBarVEmpty + vs);  // V is free once dP has read it
        if (++vs == C::kVStages) vs = 0, vph ^= 1;
      }
    } else if (warp == C::kMmaWarp + 3) {
      // ------------------------------------------------------------ warp Z: S(j) = Q K_j^T
      const uint32_t elected = elect_one();
      int ks = 0, kph = 0;  // ring position of the next K tile
      bool ok = mbar_wait_warp(bar(C::kBarQ), 0, w, kBSiteMmaQ);
      for (int j = 0; ok && j < nkv; ++j) {
        if (j >= 2) {
          // score buffer j%2 holds dS(j-2) until dQ += dS(j-2) K_(j-2) has completed
          if (!(ok = mbar_wait_warp(bar(C::kBarDqDone + (j & 1)), ((j - 2) >> 1) & 1, w, kBSiteMmaDs))) break;
          tc_fence_after();
        }
        if (!(ok = mbar_wait_warp(bar(C::kBarKFull + ks), kph, w, kBSiteMmaKV))) break;
        issue_rows_x_rows<D, BF16, W, KD>(elected, tmem_base + C::kColS + (j & 1) * W, smem_base + C::kOffQ,
                                   smem_base + C::kOffK + ks * C::kKvBytes);
        commit_to(elected, C::kBarSFull + (j & 1));
        commit_to(elected, C::kBarKEmpty + ks);
        if (++ks == C::kKStages) ks = 0, kph ^= 1;
      }
    } else if (warp == C::kMmaWarp + 2) {
      // ------------------------------------------------------------ warp Y: dQ += dS(j) K_j
      const uint32_t elected = elect_one();
      bool ok = true;
      int ks = 0, kph = 0;
      for (int j = 0; ok && j < nkv; ++j) {
        if (!(ok = mbar_wait_warp(bar(C::kBarKFull + ks), kph, w, kBSiteMmaKV))) break;
        if (!(ok = mbar_wait_warp(bar(C::kBarDsReady + (j & 1)), (j >> 1) & 1, w, kBSiteMmaDs))) break;
        tc_fence_after();
        clear_rows<D, W>(smem + C::kOffK + ks * C::kKvBytes, e.length - j * W, lane);  // S(j) has been formed
        issue_tmem_x_tile<D, BF16, W, KD>(elected, tmem_base + C::kColDQ, tmem_base + C::kColS + (j & 1) * W, kCols,
                                   smem_base + C::kOffK + ks * C::kKvBytes, j > 0);
        commit_to(elected, C::kBarDqDone + (j & 1));
        commit_to(elected, C::kBarKEmpty + ks);
        if (++ks == C::kKStages) ks = 0, kph ^= 1;
      }
      if (ok) commit_to(elected, C::kBarDone);
    }
    __syncwarp();
  } else {
    reg_inc<C::kComputeRegs>();
    const int wg = warp >> 2;
    const int w4 = warp & 3;
    const int r = w4 * 32 + lane;  // q row in the tile = tensor-memory lane
    const uint32_t lane_base = static_cast<uint32_t>(w4 * 32) << 16;
    const uint32_t tDp = tmem_base + lane_base + C::kColDp + wg * kCols;
    const float2 sc2 = make_float2(scale_log2, scale_log2);
    float inv_dscale;
    const float dscale = heads_dscale<BF16>(stats, capacity, e.base, (e.length + 127) >> 7, head, 1, lane, &inv_dscale);
    const float ds_scale = scale * dscale * kProbabilityInverse<BF16>;
    const float2 scale2 = make_float2(ds_scale, ds_scale);
    bool ok = mbar_wait_warp(bar(C::kBarQ), 0, w, kBSiteCmpQ);
    float2 nlse2 = make_float2(0.f, 0.f), ndlt2 = make_float2(0.f, 0.f);
    if (ok) {
      const float* st = reinterpret_cast<const float*>(smem + C::kOffStats);
      nlse2 = make_float2(st[r], st[r]);              // -lse*log2e of this row (+ kProbabilityPower)
      ndlt2 = make_float2(st[128 + r], st[128 + r]);  // -delta of this row
    }
    for (int j = 0; ok && j < nkv; ++j) {
      const uint32_t tS = tmem_base + lane_base + C::kColS + (j & 1) * W + wg * kCols;
      if (!(ok = mbar_wait_warp(bar(C::kBarSFull + (j & 1)), (j >> 1) & 1, w, kBSiteCmpSt))) break;
      tc_fence_after();
      float2 p[kPairs];
      {
        uint32_t sr[kCols];
#pragma unroll
        for (int c = 0; c < kCols; c += 32) tmem_ld_x32(tS + c, sr + c);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < kPairs; ++c) {
          const float2 t = __ffma2_rn(make_float2(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])), sc2, nlse2);
          p[c] = exp2_pair<kPolyShareT<D>>(t, c);
        }
      }
      if (j * W + W > qt * 128) {  // diagonal tile: keep kv <= q, which leaves out the keys behind the sequence too
        const int last = qt * 128 + r - j * W - wg * kCols;
#pragma unroll
        for (int c = 0; c < kPairs; ++c) {
          p[c].x = (2 * c <= last) ? p[c].x : 0.f;
          p[c].y = (2 * c + 1 <= last) ? p[c].y : 0.f;
        }
      }
      if (!(ok = mbar_wait_warp(bar(C::kBarDpFull), j & 1, w, kBSiteCmpDpt))) break;
      tc_fence_after();
      uint32_t dp[kCols];
#pragma unroll
      for (int c = 0; c < kCols; c += 32) tmem_ld_x32(tDp + c, dp + c);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kBarDpConsumed));
      uint32_t dsk[kPairs];
#pragma unroll
      for (int c = 0; c < kPairs; ++c) {
        float2 u = __fadd2_rn(make_float2(__uint_as_float(dp[2 * c]), __uint_as_float(dp[2 * c + 1])), ndlt2);
        u = __fmul2_rn(__fmul2_rn(p[c], u), scale2);
        dsk[c] = pack2<kInterBF16<BF16>>(u.x, u.y);
      }
      // over the score columns this thread has already read
      if constexpr (kPairs == 16) tmem_st_x16(tS, dsk); else tmem_st_x32(tS, dsk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::kBarDsReady + (j & 1)));
    }
    if (ok && wg == 0 && mbar_wait_warp(bar(C::kBarDone), 0, w, kBSiteCmpDone)) {
      tc_fence_after();
      store_packed_rows<D, BF16, KD>(tmem_base + lane_base + C::kColDQ, smem + C::kOffDO, w4, lane, &tdq, row_q + w4 * 32, head, Hq,
                                     e.length - qt * 128 - w4 * 32, dq, cols, inv_dscale);
    }
  }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  if (blockIdx.x == gridDim.x - 1) grid_wait_previous();
}

template <int D, bool BF16, int KD, int W, int S>
cudaError_t launch_dkdv_s(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                          const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk, const CUtensorMap& tdv,
                          void* dk, void* dv, const PackedStats& stats, int* status, cudaStream_t stream) {
  using C = DkdvCfg<D, 0, W>;
  auto kern = packed_dkdv_kernel<D, BF16, KD, W, S>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return e;
  return launch_dependent_cluster(kern, static_cast<unsigned>(plan.capacity) * s.Hkv * S, S, C::kThreads, C::kSmemBytes, stream, tq, tk, tv,
                                  tdo, tdk, tdv, dk, dv, plan.tiles, plan.counts, stats, plan.capacity, s.Hkv, s.Hq / s.Hkv, s.Dg, s.scale,
                                  s.scale * 1.4426950408889634f, status);
}
template <int D, bool BF16, int KD, int W>
cudaError_t launch_dkdv_t(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                          const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk, const CUtensorMap& tdv,
                          void* dk, void* dv, const PackedStats& stats, int cluster, int* status, cudaStream_t stream) {
  if constexpr (W == 128) {
    if (cluster == 4) return launch_dkdv_s<D, BF16, KD, W, 4>(s, plan, tq, tk, tv, tdo, tdk, tdv, dk, dv, stats, status, stream);
    if (cluster == 2) return launch_dkdv_s<D, BF16, KD, W, 2>(s, plan, tq, tk, tv, tdo, tdk, tdv, dk, dv, stats, status, stream);
  }
  return launch_dkdv_s<D, BF16, KD, W, 1>(s, plan, tq, tk, tv, tdo, tdk, tdv, dk, dv, stats, status, stream);
}
template <int D, bool BF16, int KD, int W>
cudaError_t launch_dq_t(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                        const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdq, void* dq, const PackedStats& stats,
                        int* status, cudaStream_t stream) {
  using C = PackedDqCfg<D, W>;
  auto kern = packed_dq_kernel<D, BF16, KD, W>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, static_cast<unsigned>(plan.capacity) * s.Hq, C::kThreads, C::kSmemBytes, stream, tq, tk, tv, tdo, tdq,
                          dq, plan.tiles, plan.counts, stats, plan.capacity, s.Hq, s.Hq / s.Hkv, s.Dg, s.scale,
                          s.scale * 1.4426950408889634f, status);
}

}  // namespace

// 64 (two CTAs on an SM) up to head dim 64, once there are CTAs to pair (DkdvCfg in bwd_roles.cuh), by the tiles that the rows
// have at most.  Whole backward, fp16, head dim 64, microseconds with the line at 100 / 200 / 300 CTAs a hundred SMs / none:
// 2 x 2048 rows, 16 / 4 heads 119 / 97 / 98 / 103, 4 x 1024 74 / 67 / 66 / 74, 32 x 300, 8 / 2 heads 62 / 60 / 67 / 79.
int packed_step_rows(const PackedShape& s, int heads, int num_sms) {
  return s.D <= 64 && 100ll * packed_capacity(s.rows, s.batch) * heads >= 200ll * num_sms ? 64 : 128;
}

// Four where there are very few CTAs, two where there are few, or about as many as SMs for long sequences, whose heaviest tiles the dQ kernel cannot fill up behind.
// Forward and backward replayed, bf16, microseconds, single CTAs / clusters, by CTAs for each SM:
//   head dim 128, 8 / 2 heads: 8 x 512 rows (0.54) 61.2 / 61.1, 16 x 256 (0.65) 49.3 / 53.3, 4 x 1024 (0.49) 88.4 / 74.6, 8 x 1024 (0.97) 112.6 / 120.6,
//   2 x 2048 (0.46) 146 / 105, 4 x 2048 (0.92) 158 / 166, 2 x 4096 (0.89) 268 / 264, 16 x 512 (1.08) 89 / 97.5; 2 x 8192, 8 / 1 (0.88) 1128 / 1041,
//   2 x 2048, 32 / 1 (0.23) 837 / 462, clusters of four 293, 4096, 8 / 1 (0.22) 257 of two / 170 of four, 2 x 1024, 8 / 2 (0.24) 61.6 / 55.2,
//   16 x 200, 32 / 1 (0.28) 128 / 129;   head dim 64: 4096, 16 / 4 (0.89) 234 / 205, eight of 256 to 1024, 16 / 4 (0.92) 62.2 / 66.7.
int packed_cluster(const PackedShape& s, int num_sms) {
  const long long ctas = static_cast<long long>(packed_capacity(s.rows, s.batch)) * s.Hkv;
  if (s.Hq / s.Hkv % 4 == 0 && 4 * ctas <= num_sms) return 4;
  return s.Hq / s.Hkv % 2 == 0 && (2 * ctas <= num_sms || (ctas <= num_sms && s.rows >= 4096ll * s.batch)) ? 2 : 1;
}

#define FA2_DTYPES(CALL, DD, KK, WW) return s.dtype ? CALL<DD, true, KK, WW>(FA2_ARGS) : CALL<DD, false, KK, WW>(FA2_ARGS)
#define FA2_DISPATCH(CALL)                                        \
  if (s.D == 32 && step_rows == 64) FA2_DTYPES(CALL, 32, 32, 64); \
  if (s.D == 64 && step_rows == 64) FA2_DTYPES(CALL, 64, 64, 64); \
  if (s.D == 32) FA2_DTYPES(CALL, 32, 32, 128);                   \
  if (s.D == 64) FA2_DTYPES(CALL, 64, 64, 128);                   \
  if (s.Dg <= kShortDim128) FA2_DTYPES(CALL, 128, kShortDim128, 128); \
  FA2_DTYPES(CALL, 128, 128, 128)

cudaError_t launch_packed_dkdv(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                               const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk, const CUtensorMap& tdv,
                               void* dk, void* dv, const PackedStats& stats, int step_rows, int cluster, int* status, cudaStream_t stream) {
#define FA2_ARGS s, plan, tq, tk, tv, tdo, tdk, tdv, dk, dv, stats, cluster, status, stream
  FA2_DISPATCH(launch_dkdv_t);
#undef FA2_ARGS
}

cudaError_t launch_packed_dq(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                             const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdq, void* dq,
                             const PackedStats& stats, int step_rows, int* status, cudaStream_t stream) {
#define FA2_ARGS s, plan, tq, tk, tv, tdo, tdq, dq, stats, status, stream
  FA2_DISPATCH(launch_dq_t);
#undef FA2_ARGS
}
#undef FA2_DISPATCH
#undef FA2_DTYPES

}  // namespace fa2
