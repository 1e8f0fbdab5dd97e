// Causal attention forward over packed sequences with grouped heads (packed.cuh).
//
// The arithmetic, the warp roles and the tensor-memory plan are those of fwd_kernel (fwd.cu) with 128-row KV tiles:
// a CTA has two score tiles in turn on one buffer, a softmax group for each, and two MMA-issuing warps.  What differs is the work
// item.  Its two Q tiles are the same rows of two query heads that share a key head, so they read each K and V tile
// once, end at the same KV tile, and a sequence of one tile still fills both.  With an odd number G of query heads to a
// key head the 2 G (tile, head) of two adjacent tiles make G items; one of them has either tile.  The items come from the plan, heaviest first, all heads of a tile
// one after the other (their K and V pass the L2 together).  Bound by the chain of a softmax step at head dim 128, by the
// exponentials below, like fwd_kernel.  P enters the second product in 16 bits, the type that the tensor pipe takes beside V (fp16: as P 2^11,
// kWeightPower): the output's error is 1.2 to 1.3 times that of its own rounding.  Sums and the output before its one rounding are fp32.
// bf16, 8 808 rows in six sequences, 32 / 8 heads of 128 columns: 158 us a call in a burst (1 130 TFLOP/s, tensor pipe 63 % active), 187 in
// a long loop, at the power limit.
#include "mma_issue.cuh"
#include "packed.cuh"

namespace fa2 {
namespace {

constexpr int kThreads = 384;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct PackedFwdCfg {
  using T = Tile<D>;
  static constexpr int kPolyShare = D == 32 ? 3 : 0;  // as FwdCfg
  static constexpr float kRescaleThreshold = 8.0f;  // as FwdCfg: 4 at fp16
  static constexpr int kLaunchRegs = 65536 / kThreads / 8 * 8;
  static constexpr int kProducerRegs = 72;
  static constexpr int kSoftmaxRegs = 216;
  static_assert(128 * kProducerRegs + 256 * kSoftmaxRegs <= kThreads * kLaunchRegs,
                "setmaxnreg.inc waits for registers that setmaxnreg.dec has released");
  static constexpr int kStages = D == 128 ? 2 : 4;  // of the K ring and of the V ring
  static constexpr int kStageBytes = 32 * T::kRowBytes;  // output staging of one softmax warp
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + 2 * T::kTileBytes;
  static constexpr int kOffV = kOffK + kStages * T::kTileBytes;
  static constexpr int kOffStage = kOffV + kStages * T::kTileBytes;
  static constexpr int kOffBar = kOffStage + 8 * kStageBytes;
  static constexpr int kBarItemFull = 0;   // 2: the work item in slot n % 2 may be read
  static constexpr int kBarItemEmpty = 2;  // 2: every role but the producer has read it (10 arrivals)
  static constexpr int kBarQFull = 4;
  static constexpr int kBarQEmpty = 5;     // the item's last score product has read the Q tiles
  static constexpr int kBarKFull = 6;
  static constexpr int kBarKEmpty = kBarKFull + kStages;
  static constexpr int kBarVFull = kBarKEmpty + kStages;
  static constexpr int kBarVEmpty = kBarVFull + kStages;
  static constexpr int kBarSFull = kBarVEmpty + kStages;  // 2: S holds slot i's scores
  static constexpr int kBarSFree = kBarSFull + 2;         // 2: group i has copied S out (4 arrivals)
  static constexpr int kBarPFull = kBarSFree + 2;         // 2: P_i written, O_i rescaled (4 arrivals)
  static constexpr int kBarPvDone = kBarPFull + 2;        // 2: O_i += P_i V completed
  static constexpr int kNumBars = kBarPvDone + 2;
  static constexpr int kOffItems = (kOffBar + kNumBars * 8 + 15) / 16 * 16;  // 2 items of 32 bytes
  static constexpr int kSmemBytes = kOffItems + 2 * 32 + 16;                 // + tmem slot, abort flag, next item
  static constexpr int kColS = 0, kColP = 128, kColO = 256;
  static_assert(kColO + 2 * D <= 512, "tensor memory");
  static_assert(kSmemBytes + 1024 <= 228 * 1024, "shared memory of one SM");
};

struct PackedItem {
  int row0, length;  // length 0: no more items
  int tile[2];       // tile[1] < 0: there is no second one
  int head[2];
  int pad[2];
};
static_assert(sizeof(PackedItem) == 32, "item slots");

enum Site { kSiteLoadK = 128, kSiteLoadV, kSiteMmaQ, kSiteMmaK, kSiteMmaV, kSiteMmaP, kSiteMmaSFree, kSiteSoftS, kSiteSoftPv,
            kSiteSoftO, kSiteAlign, kSiteItem, kSiteLoadQ };

template <int D, bool BF16, int KD>
__global__ void __launch_bounds__(kThreads, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to, uint16_t* out, float* lse,
                      const int* cu_seqlens, const __grid_constant__ PackedPlan plan, bool alone, int rows, int batch, int Hq, int G,
                      int cols, bool two_heads, float scale_log2, int* status) {
  using C = PackedFwdCfg<D>;
  using T = Tile<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  // Roles as in fwd_kernel: hardware warps 0-3 are 8 (S), 9 (producer), 10 (P V) and an idle one, 4-11 the softmax warps 0-7.
  const int warp = ((threadIdx.x >> 5) + 8) % 12;
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  if (smem_base & 1023u) {  // swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) atomicCAS(status, 0, 0x20000 | kSiteAlign);
    return;
  }
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffItems + 2 * sizeof(PackedItem));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* next_slot = reinterpret_cast<volatile int*>(tmem_slot + 2);
  auto bar = [&](int i) { return smem_base + C::kOffBar + 8u * i; };
  // KV tiles of slot i: those up to its diagonal
  auto kv_tiles = [&](const PackedItem& item, int i) { return item.tile[i] + 1; };

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(C::kBarItemFull + i), 1);
      mbar_init(bar(C::kBarItemEmpty + i), 10);
      mbar_init(bar(C::kBarSFull + i), 1);
      mbar_init(bar(C::kBarSFree + i), 4);
      mbar_init(bar(C::kBarPFull + i), 4);
      mbar_init(bar(C::kBarPvDone + i), 1);
    }
    mbar_init(bar(C::kBarQFull), 1);
    mbar_init(bar(C::kBarQEmpty), 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(bar(C::kBarKFull + i), 1);
      mbar_init(bar(C::kBarKEmpty + i), 1);
      mbar_init(bar(C::kBarVFull + i), 1);
      mbar_init(bar(C::kBarVEmpty + i), 1);
    }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const WaitCtx w{abort_flag, status};
  grid_wait_previous();
  grid_allow_next();

  // Slot of the n-th item of this CTA, for every role but the producer; false: there is none, or the CTA gives up.
  // It votes; the other waits of the warp that issues S do not, see fwd_kernel.
  auto take_item = [&](int n, PackedItem& item) {
    if (!mbar_wait_warp(bar(C::kBarItemFull + (n & 1)), (n >> 1) & 1, w, kSiteItem)) return false;
    item = reinterpret_cast<const PackedItem*>(smem + C::kOffItems)[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(C::kBarItemEmpty + (n & 1)));
    return item.length > 0;
  };

  if (warp >= 8) {
    reg_dec<C::kProducerRegs>();
    if (warp == 9) {
      // ---------------------------------------------------------------- draws the items; TMA producer
      const uint32_t elected = elect_one();
      if (elected) {
        prefetch_tensormap(&tq);
        prefetch_tensormap(&tk);
        prefetch_tensormap(&tv);
      }
      const int per_tile = two_heads ? Hq / 2 : Hq;  // items of a list entry
      const PackedTile* const list = two_heads ? plan.tiles : plan.pairs;
      const int per = two_heads ? 1 : 2;  // tiles of an entry
      // alone: this lane's sequence, and the entries it has in the list that there is no plan of
      int start = 0, length = 0, mine = 0, entries;
      if (alone) {
        const ShortBatch s(cu_seqlens, batch, rows);
        start = s.start, length = s.length, mine = ((s.length + 127) / 128 + per - 1) / per;
        entries = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(mine));
      } else {
        entries = ld_global(plan.counts + (two_heads ? 0 : 1));
      }
      const int total_items = entries * per_tile;
      // Entry `at` of that list, which has the order of write_list_by_ballots (whole warp).
      auto find = [&](int at) {
        auto from = [&](int number) { return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(max(mine - number, 0)))); };
        int low = 0, high = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(mine)));
        while (low + 1 < high) {
          const int mid = (low + high) >> 1;
          if (from(mid) > at) low = mid; else high = mid;
        }
        const int rank = at - from(low + 1);  // among the sequences that have an entry of number `low`
        const unsigned same = __ballot_sync(0xffffffffu, mine > low);
        const int l = __ffs(__ballot_sync(0xffffffffu, mine > low && __popc(same & ((1u << lane) - 1u)) == rank)) - 1;
        return PackedTile{__shfl_sync(0xffffffffu, start, l), __shfl_sync(0xffffffffu, length, l), low * per, 0};
      };
      bool ok = true;
      int ks = 0, kph = 0, vs = 0, vph = 0;  // ring positions
      int drawn = blockIdx.x;                // an item, or total_items or more: there is none
      const bool draws = !alone && total_items > static_cast<int>(gridDim.x);
      int round = 0;
      auto draw = [&]() {
        if (alone)  // to and fro through the list, so that who has the heaviest of one round has the lightest of the next
          ++round, drawn = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        else if (lane == 0)
          drawn = draws ? atomicAdd(plan.counts + 2, 1) : total_items;
      };
      auto drawn_item = [&]() {  // the number drawn, for the whole warp
        if (lane == 0) *next_slot = drawn;
        __syncwarp();
        const int id = *next_slot;
        __syncwarp();
        return id;
      };
      if (draws) draw();
      for (int n = 0;; ++n) {
        const int id = drawn_item();
        PackedItem item{0, 0, {-1, -1}, {0, 0}, {0, 0}};
        if (id < total_items) {
          const int entry = id / per_tile, h = id - entry * per_tile;
          const PackedTile e = alone ? find(entry) : load_tile(list + entry);
          if (two_heads) {
            item = PackedItem{e.row0, e.length, {e.tile, e.tile}, {2 * h, 2 * h + 1}, {0, 0}};
          } else {
            // the two of number x and x + 1 among the (tile, head) of the entry and key head, tile by tile
            const int kv_head = h / G, x = 2 * (h - kv_head * G), there = e.tile * 128 + 128 < e.length ? 2 * G : G;
            if (x >= there) {  // the entry has one tile, and the items before this one have taken it
              draw();
              --n;
              continue;
            }
            const int t0 = x >= G, t1 = x + 1 >= G, head = kv_head * G + x;
            item = PackedItem{e.row0, e.length, {e.tile + t0, x + 1 < there ? e.tile + t1 : -1}, {head - t0 * G, head + 1 - t1 * G}, {0, 0}};
          }
        }
        if (ok) ok = mbar_wait_warp(bar(C::kBarItemEmpty + (n & 1)), ((n >> 1) & 1) ^ 1, w, kSiteItem);
        if (ok && lane == 0) {
          reinterpret_cast<PackedItem*>(smem + C::kOffItems)[n & 1] = item;
          mbar_arrive(bar(C::kBarItemFull + (n & 1)));
        }
        if (item.length == 0) break;
        const HeadCoord hk{item.head[0] / G, 0};
        const int nkv = max(kv_tiles(item, 0), kv_tiles(item, 1));
        bool asked = false;  // the next item's number has been drawn
        // K runs one KV tile ahead of V: S(j+1) is issued during KV step j
        for (int t = 0; ok && t <= nkv; ++t) {
          if (t < nkv) {
            if (!(ok = mbar_wait_warp(bar(C::kBarKEmpty + ks), kph ^ 1, w, kSiteLoadK))) break;
            if (elected) {
              mbar_arrive_expect_tx(bar(C::kBarKFull + ks), T::kTileBytes);
#pragma unroll
              for (int ch = 0; ch < T::kChunks; ++ch)
                tma_load_4d(smem_base + C::kOffK + ks * T::kTileBytes + ch * T::kChunkTileBytes, &tk, ch * T::kChunkElems,
                            item.row0 + t * 128, hk, bar(C::kBarKFull + ks));
            }
            if (++ks == C::kStages) ks = 0, kph ^= 1;
          }
          if (t == 0) {
            if (!(ok = mbar_wait_warp(bar(C::kBarQEmpty), (n & 1) ^ 1, w, kSiteLoadQ))) break;
            if (elected) {
              const int slots = item.tile[1] >= 0 ? 2 : 1;
              mbar_arrive_expect_tx(bar(C::kBarQFull), slots * T::kTileBytes);
              for (int i = 0; i < slots; ++i)
                for (int ch = 0; ch < T::kChunks; ++ch)
                  tma_load_4d(smem_base + C::kOffQ + i * T::kTileBytes + ch * T::kChunkTileBytes, &tq, ch * T::kChunkElems,
                              item.row0 + item.tile[i] * 128, HeadCoord{item.head[i], 0}, bar(C::kBarQFull));
            }
          }
          if (t >= 1) {
            if (t == nkv) {
              asked = true;
              draw();
            }
            if (!(ok = mbar_wait_warp(bar(C::kBarVEmpty + vs), vph ^ 1, w, kSiteLoadV))) break;
            if (elected) {
              mbar_arrive_expect_tx(bar(C::kBarVFull + vs), T::kTileBytes);
#pragma unroll
              for (int ch = 0; ch < T::kChunks; ++ch)
                tma_load_4d(smem_base + C::kOffV + vs * T::kTileBytes + ch * T::kChunkTileBytes, &tv, ch * T::kChunkElems,
                            item.row0 + (t - 1) * 128, hk, bar(C::kBarVFull + vs));
            }
            if (++vs == C::kStages) vs = 0, vph ^= 1;
          }
        }
        if (!asked) draw();
      }
    } else if (warp == 8) {
      // ---------------------------------------------------------------- S = Q_i K_j^T issuer
      const uint32_t elected = elect_one();
      auto commit = [&](int b) {
        if (elected) mma_commit(bar(b));
      };
      bool ok = true;
      int ks = 0, kph = 0;           // K ring position
      int prev_i = -1, prev_ph = 0;  // group and phase of the previous score product
      int count[2] = {0, 0};         // score products of either group so far
      PackedItem item;
      for (int n = 0; ok && take_item(n, item); ++n) {
        const int n0 = kv_tiles(item, 0), n1 = kv_tiles(item, 1), nkv = max(n0, n1);
        ok = mbar_wait(bar(C::kBarQFull), n & 1, w, kSiteMmaQ);
        for (int j = 0; ok && j < nkv; ++j) {
          if (!(ok = mbar_wait(bar(C::kBarKFull + ks), kph, w, kSiteMmaK))) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (j >= (i == 0 ? n0 : n1)) continue;
            if (prev_i >= 0) {
              if (!(ok = mbar_wait(bar(C::kBarSFree + prev_i), prev_ph, w, kSiteMmaSFree))) break;
              tc_fence_after();
            }
            const bool last_of_tile = i == 1 || n1 == 0;
            issue_rows_x_rows<D, BF16, 128, KD>(elected, tmem_base + C::kColS, smem_base + C::kOffQ + i * T::kTileBytes,
                                                smem_base + C::kOffK + ks * T::kTileBytes);
            if (last_of_tile) {
              commit(C::kBarKEmpty + ks);  // both products that read K_j issued
              if (++ks == C::kStages) ks = 0, kph ^= 1;
              if (j == nkv - 1) commit(C::kBarQEmpty);
            }
            commit(C::kBarSFull + i);
            prev_i = i;
            prev_ph = count[i]++ & 1;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
    } else if (warp == 10) {
      // ---------------------------------------------------------------- O_i += P_i V_j issuer
      const uint32_t elected = elect_one();
      auto commit = [&](int b) {
        if (elected) mma_commit(bar(b));
      };
      bool ok = true;
      int vs = 0, vph = 0;    // V ring position
      int count[2] = {0, 0};  // products of either group so far
      PackedItem item;
      for (int n = 0; ok && take_item(n, item); ++n) {
        const int n0 = kv_tiles(item, 0), n1 = kv_tiles(item, 1), nkv = max(n0, n1);
        for (int j = 0; ok && j < nkv; ++j) {
          // the waits of this warp vote: clear_rows wants it converged
          if (!(ok = mbar_wait_warp(bar(C::kBarVFull + vs), vph, w, kSiteMmaV))) break;
          clear_rows<D, 128>(smem + C::kOffV + vs * T::kTileBytes, item.length - j * 128, lane);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (j >= (i == 0 ? n0 : n1)) continue;
            if (!(ok = mbar_wait_warp(bar(C::kBarPFull + i), count[i]++ & 1, w, kSiteMmaP))) break;
            tc_fence_after();
            issue_tmem_x_tile<D, BF16, 128, KD>(elected, tmem_base + C::kColO + i * D, tmem_base + C::kColP + i * 64, 32,
                                                smem_base + C::kOffV + vs * T::kTileBytes, j > 0);
            if (i == 1 || n1 == 0) {
              commit(C::kBarVEmpty + vs);
              if (++vs == C::kStages) vs = 0, vph ^= 1;
            }
            commit(C::kBarPvDone + i);
          }
        }
      }
    } else if (alone) {
      // ---------------------------------------------------------------- warp 11, where there is no plan kernel
      const ShortBatch s(cu_seqlens, batch, rows);
      if (blockIdx.x == 0) write_short_plan(s, plan, !two_heads, 0, 1, status);
      clear_outside(out, static_cast<long long>(Hq) * cols / 8, s.first, s.last, rows, blockIdx.x * 32ll + lane, gridDim.x * 32ll);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax groups
    reg_inc<C::kSoftmaxRegs>();
    const int wg = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row inside the Q tile = tensor-memory lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + lane_base + C::kColS;
    const uint32_t tP = tmem_base + lane_base + C::kColP + wg * 64;
    const uint32_t tO = tmem_base + lane_base + C::kColO + wg * D;
    bool ok = true;
    int done = 0;  // KV tiles of this group's earlier items
    PackedItem item;
    for (int n = 0; ok && take_item(n, item); ++n) {
      const int qt = wg == 0 ? item.tile[0] : item.tile[1], head = wg == 0 ? item.head[0] : item.head[1];
      const int nj = qt + 1;
      const int local = qt * 128 + (warp & 3) * 32;  // first row of this warp in the sequence
      const bool mine = local + lane < item.length;
      // rows behind the sequence ask for no rescale, so that what they hold changes no bit of the others
      const float threshold = mine ? weight_lag<BF16>(C::kRescaleThreshold) : INFINITY;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < nj; ++j) {
        const int ph = (done + j) & 1;  // of this tile on the group's barriers
        if (!(ok = mbar_wait_warp(bar(C::kBarSFull + wg), ph, w, kSiteSoftS))) break;
        tc_fence_after();
        uint32_t sr[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld_x32(tS + c, sr + c);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kBarSFree + wg));  // S may be overwritten now
        float* s = reinterpret_cast<float*>(sr);
        if (j == qt) {  // diagonal tile: keep col <= row, which leaves out the rows behind the sequence too
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = (c <= r) ? s[c] : -INFINITY;
        }
        float mx[4];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          mx[q4] = max3(s[32 * q4], s[32 * q4 + 1], s[32 * q4 + 2]);
#pragma unroll
          for (int c = 3; c < 31; c += 2) mx[q4] = max3(mx[q4], s[32 * q4 + c], s[32 * q4 + c + 1]);
          mx[q4] = fmaxf(mx[q4], s[32 * q4 + 31]);
        }
        const float m_new = fmaxf(max3(m_run, mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool need = (m_new - m_run) * scale_log2 > threshold;
        bool pv_waited = false;
        if (__any_sync(0xffffffffu, need)) {
          // A neighbour's rescale must not touch a row without a finite score so far: -inf - -inf is no factor.
          const float alpha = m_new == -INFINITY ? 1.0f : ex2((m_run - m_new) * scale_log2);
          l_run *= alpha;
          m_run = m_new;
          if (j > 0) {
            // O_i must be at rest: wait for O_i += P_i(j-1) V_(j-1)
            if (!(ok = mbar_wait_warp(bar(C::kBarPvDone + wg), ph ^ 1, w, kSiteSoftPv))) break;
            tc_fence_after();
            pv_waited = true;
#pragma unroll
            for (int c0 = 0; c0 < KD; c0 += 32) {
              uint32_t orr[32];
              tmem_ld_x32(tO + c0, orr);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) orr[c] = __float_as_uint(__uint_as_float(orr[c]) * alpha);
              tmem_st_x32(tO + c0, orr);
            }
          }
        }
        // p = 2^(s*c - m*c) with packed fp32x2 FMAs; row sum in four independent packed chains
        const float2 sc2 = make_float2(scale_log2, scale_log2);
        // a row whose scores so far are all -inf has weights 0; its first finite score rescales them away
        const float neg_m = m_run == -INFINITY ? 0.f : kWeightPower<BF16> - m_run * scale_log2;
        const float2 nm2 = make_float2(neg_m, neg_m);
        float2 acc[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        uint32_t pk[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) {
          float2 t = __ffma2_rn(make_float2(s[2 * c], s[2 * c + 1]), sc2, nm2);
          if ((c & 7) < C::kPolyShare) {
            t = ex2_poly2(t);
          } else {
            t.x = ex2(t.x);
            t.y = ex2(t.y);
          }
          acc[c & 3] = __fadd2_rn(acc[c & 3], t);
          pk[c] = pack2<kInterBF16<BF16>>(t.x, t.y);
        }
        if (j > 0 && !pv_waited) {
          // P_i still feeds O_i += P_i(j-1) V_(j-1) until that product has completed
          if (!(ok = mbar_wait_warp(bar(C::kBarPvDone + wg), ph ^ 1, w, kSiteSoftPv))) break;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 32) tmem_st_x32(tP + c, pk + c);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(C::kBarPFull + wg));
        const float2 a01 = __fadd2_rn(acc[0], acc[1]), a23 = __fadd2_rn(acc[2], acc[3]);
        l_run += (a01.x + a01.y) + (a23.x + a23.y);
      }
      done += nj;
      if (ok && nj > 0 && (ok = mbar_wait_warp(bar(C::kBarPvDone + wg), (done - 1) & 1, w, kSiteSoftO))) {
        tc_fence_after();
        // a row without any finite score has no softmax, whatever weights it was left with
        const float inv_l = m_run == -INFINITY ? __uint_as_float(0x7fffffffu) : 1.0f / l_run;
        const bool whole = local + 32 <= item.length;
        const HeadCoord hc{head, 0};
        const long long row = item.row0 + local + lane;
        uint8_t* const sO = smem + C::kOffStage + warp * C::kStageBytes;
#pragma unroll
        for (int c0 = 0; c0 < KD; c0 += 32) {
          uint32_t orr[32];
          tmem_ld_x32(tO + c0, orr);
          tmem_wait_ld();
          const int piece0 = (c0 % T::kChunkElems) / 8;
          if (piece0 == 0) {
            // the staging piece may be refilled once the store before has READ it
            if (lane == 0) tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            uint4 val;
            val.x = pack2<BF16>(__uint_as_float(orr[8 * p + 0]) * inv_l, __uint_as_float(orr[8 * p + 1]) * inv_l);
            val.y = pack2<BF16>(__uint_as_float(orr[8 * p + 2]) * inv_l, __uint_as_float(orr[8 * p + 3]) * inv_l);
            val.z = pack2<BF16>(__uint_as_float(orr[8 * p + 4]) * inv_l, __uint_as_float(orr[8 * p + 5]) * inv_l);
            val.w = pack2<BF16>(__uint_as_float(orr[8 * p + 6]) * inv_l, __uint_as_float(orr[8 * p + 7]) * inv_l);
            if (whole)
              *reinterpret_cast<uint4*>(sO + swizzled_offset<D>(lane, piece0 + p)) = val;
            else if (mine && c0 + 8 * p < cols)
              *reinterpret_cast<uint4*>(out + (row * Hq + head) * cols + c0 + 8 * p) = val;
          }
          if (whole && ((c0 + 32) % T::kChunkElems == 0 || c0 + 32 == KD)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_4d(&to, c0 / T::kChunkElems * T::kChunkElems, item.row0 + local, hc, smem_u32(sO));
              tma_store_commit();
            }
          }
        }
        tc_fence_before();  // O_i is overwritten by the next item's first product, which this group's P lets in
        if (mine) lse[static_cast<size_t>(head) * rows + row] = (m_run * scale_log2 + lg2(l_run * kWeightInverse<BF16>)) * kLn2;
      }
    }  // items
    if (lane == 0) tma_store_wait_read();
  }

  // ---------------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Work items at most.
long long most_items(const PackedShape& s) {
  return static_cast<long long>(packed_capacity(s.rows, s.batch)) * (s.Hq / s.Hkv % 2 == 0 ? s.Hq / 2 : s.Hq);
}

template <int D, bool BF16, int KD = D>
cudaError_t launch_t(const PackedShape& s, const int* cu_seqlens, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                     const CUtensorMap& tv, const CUtensorMap& to, void* out, float* lse, int* status, int num_sms, cudaStream_t stream) {
  using C = PackedFwdCfg<D>;
  auto kern = packed_fwd_kernel<D, BF16, KD>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return e;
  const bool two_heads = s.Hq / s.Hkv % 2 == 0;
  const long long items = most_items(s);
  const unsigned grid = static_cast<unsigned>(items < num_sms ? items : num_sms);
  return launch_dependent(kern, grid, kThreads, C::kSmemBytes, stream, tq, tk, tv, to, static_cast<uint16_t*>(out), lse, cu_seqlens, plan,
                          packed_fwd_alone(s, num_sms), s.rows, s.batch, s.Hq, s.Hq / s.Hkv, s.Dg, two_heads,
                          s.scale * 1.4426950408889634f, status);
}

}  // namespace

// Up to 32 sequences (a warp looks through them) and a few items to a CTA: who finds items alone cannot draw them, and takes a fixed share.
// Microseconds with the plan / alone: 16 x 200 rows, 8 / 8 heads of 64 (2.2 items a CTA) 11.5 / 9.7, 4 x 512, 16 / 4 (1.1) 14.1 / 12.7,
// eight of 256 to 1024, 16 / 4 (2.5) 25.1 / 24.9, 8 x 1024, 8 / 8 (3.9) 25.6 / 23.6, 32 x 300, 16 / 4 (5.8) 33.4 / 35.7,
// six of 616 to 4096, 32 / 8 of 128 (8) 160 / 163.
constexpr int kAloneRounds = 4;
bool packed_fwd_alone(const PackedShape& s, int num_sms) { return s.batch <= 32 && most_items(s) <= kAloneRounds * num_sms; }

cudaError_t launch_packed_fwd(const PackedShape& s, const int* cu_seqlens, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                              const CUtensorMap& tv, const CUtensorMap& to, void* out, float* lse, int* status, int num_sms,
                              cudaStream_t stream) {
#define FA2_CASE(DD, KK)                                                                          \
  return s.dtype ? launch_t<DD, true, KK>(s, cu_seqlens, plan, tq, tk, tv, to, out, lse, status, num_sms, stream)  \
                 : launch_t<DD, false, KK>(s, cu_seqlens, plan, tq, tk, tv, to, out, lse, status, num_sms, stream)
  if (s.D == 32) FA2_CASE(32, 32);
  if (s.D == 64) FA2_CASE(64, 64);
  if (s.Dg <= kShortDim128) FA2_CASE(128, kShortDim128);
  FA2_CASE(128, 128);
#undef FA2_CASE
}

}  // namespace fa2
