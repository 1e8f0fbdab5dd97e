// Attention of one new token a sequence over its pages of a key-value cache.
//
//     out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),  j < lengths[b]
//
// Bound by reading the keys and values once.  The keys of every (sequence, key head) are cut into units of 64; all
// units of the call stand in one row, with room for kEnd more behind those of each (sequence, key head) for what its end costs, and
// each CTA takes an equal stretch of it, whatever the lengths are, so one long sequence and many short ones both keep
// every SM reading.  Where a stretch cuts a (sequence, key head)
// apart, each CTA leaves (m, l, o) of its part in the workspace, and decode_join_kernel adds the parts up in order:
// the same bits every time.  Where a key head has more query heads than one pass takes, neighbouring CTAs take the same
// stretch with 16 of them each, at the same time, so that the L2 serves all but the first.
//
// Inside a CTA warp w takes keys 16 w .. 16 w + 15 of every unit and runs on its own: tiled copies bring its keys and
// values into a ring of stages of its own, as many rows to a copy as 16 keys have next to each other in a page (16 where
// the page size is a multiple of it); where that is one row, the lanes bring 16 bytes each.  The keys are the 16 rows of m16n8k16 products and the query heads of the key
// head their 8 columns: S^T = K Q^T, O^T += V^T P^T, fp32 accumulators in registers, P^T turned around by
// movmatrix.  Eight query heads fill the product; as its rows they would fill half of it.  The four warps meet
// where a (sequence, key head) ends, while their next stages are already loading.  The products take a fraction of
// the time that the bytes take, so mma.sync serves, and a row of eight queries needs no tile of 128.
// 128 sequences of 500 to 8192 keys (344 905 in all), 32 / 8 heads of 128 columns, pages of 16: 231 to 244 us, 88 to 93 % of the measured copy
// rate.  Two sequences of 100 000 to 131 072, 16 / 2 heads of 128, pages of 64: 53.5 us, 47 of them decode_kernel (5.6 TB/s).
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace fa2 {
namespace {

constexpr int kUnit = 64;  // keys
// Units that the end of a (sequence, key head) counts for.  16 sequences of 8192 keys beside 500 of 100, 32 / 8 heads of 128
// columns, microseconds with 0 / 2 / 4: 161 / 146 / 171; sequences of like lengths do not mind.
constexpr int kEnd = 2;
constexpr int kWarps = 4;
constexpr int kJoinRows = 8;  // query heads that the warps of a CTA add up at a time
// Query heads of a key head that one pass takes: 8 for each column tile of the products.
inline int column_tiles(int group) { return group <= 8 ? 1 : 2; }
// Key heads that one pass takes.  Up to head dim 64 two: a warp's copies are twice as large then, and rows of 128 bytes that lie
// beside each other are read at the same time.
inline int heads_at_once(int Hkv, int D) { return D <= 64 && Hkv % 2 == 0 ? 2 : 1; }
constexpr int kMaxCtas = 1024;

template <int DP, int HP>
struct DecodeCfg {
  static_assert(HP == 1 || DP == 64, "two heads up to head dim 64");
  static constexpr int kWide = DP * HP;             // columns of a stage's row
  static constexpr int kStages = kWide == 64 ? 4 : 3;
  static constexpr int kCtasPerSm = kWide == 64 ? 3 : (kWide == 128 ? 2 : 1);
  static constexpr int kChunks = kWide / 64;        // of 64 columns, what a box of a copy is wide
  static constexpr int kTileBytes = 16 * kWide * 2; // 16 keys, or 16 values: [kChunks][16 rows][128 bytes], swizzled
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kJoinStride = DP + 4;        // floats of a row of partial sums
  static constexpr int kOffJoin = kWarps * kWarpBytes;
  static constexpr int kOffBar = kOffJoin + kWarps * kJoinRows * (kJoinStride + 2) * 4;
  static constexpr int kOffAbort = kOffBar + kWarps * kStages * 8;
  static constexpr int kSmemBytes = kOffAbort + 16;
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory of one SM");
};

// One (sequence, key head) of the call, or two key heads up to head dim 64 (HP), and the walk over the units of a CTA's stretch.
struct Walk {
  int b, h;    // the sequence; the number of the head, or pair of heads
  int unit;    // of it
  int units;   // of the sequence
  int length;  // keys of the sequence
  int left;    // of the stretch, this unit included; 0 or less: there is none
};

__device__ __forceinline__ int clamp_length(const DecodeArgs& a, int b) {
  const long long most = static_cast<long long>(a.table_width) * a.page_size;
  const long long n = ld_global(a.lengths + b);
  return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
}
__device__ __forceinline__ int units_of(int length) { return (length + kUnit - 1) / kUnit; }
__device__ __forceinline__ int room_of(int length) { return length > 0 ? units_of(length) + kEnd : 0; }

// Length of the row (whole warp).
__device__ __forceinline__ long long row_length(const DecodeArgs& a, int heads, int lane) {
  long long sum = 0;
  for (int i = 0; i < a.batch; i += 32) {
    const unsigned u = i + lane < a.batch ? room_of(clamp_length(a, i + lane)) : 0;
    sum += __reduce_add_sync(0xffffffffu, u);
  }
  return sum * heads;
}

__device__ __forceinline__ long long stretch_start(long long total, int stretch, int stretches) { return total * stretch / stretches; }

__device__ __forceinline__ void next_segment(const DecodeArgs& a, int heads, Walk& w) {
  w.unit = 0;
  if (++w.h < heads) return;
  w.h = 0;
  do {
    w.length = ++w.b < a.batch ? clamp_length(a, w.b) : 1;
    w.units = units_of(w.length);
  } while (w.units == 0);
}
__device__ __forceinline__ void next_unit(const DecodeArgs& a, int heads, Walk& w) {
  --w.left;
  if (++w.unit < w.units) return;
  w.left -= kEnd;
  if (w.left > 0) next_segment(a, heads, w);
}

// Puts `w` on the first unit of the stretch that begins at `at` of the row (whole warp); `at` is less than the row's length.
__device__ __forceinline__ void find_unit(const DecodeArgs& a, int heads, long long at, int lane, Walk& w) {
  for (int i = 0;; i += 32) {
    const int n = i + lane < a.batch ? clamp_length(a, i + lane) : 0;
    const unsigned mine = room_of(n);
    const long long all = static_cast<long long>(__reduce_add_sync(0xffffffffu, mine)) * heads;
    if (at >= all && i + 32 < a.batch) {
      at -= all;
      continue;
    }
    unsigned upto = mine;  // inclusive sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned in = __ballot_sync(0xffffffffu, static_cast<long long>(upto) * heads > at);
    const int l = __ffs(in) - 1;
    const int room = __shfl_sync(0xffffffffu, mine, l);
    w.b = i + l;
    w.units = room - kEnd;
    w.length = __shfl_sync(0xffffffffu, n, l);
    const int rest = static_cast<int>(at - static_cast<long long>(__shfl_sync(0xffffffffu, upto - mine, l)) * heads);
    w.h = rest / room;
    w.unit = rest - w.h * room;
    break;
  }
  if (w.unit >= w.units) {  // in the room behind the units
    w.left -= w.units + kEnd - w.unit;
    if (w.left > 0) next_segment(a, heads, w);
  }
}

__device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// What a part with maximum m and sum l counts beside the maximum `top` of all of them.  A part without a finite score has
// l = 0, or NaN where a score was NaN.
__device__ __forceinline__ float part_weight(float m, float l, float top, float scale_log2) {
  return m == -INFINITY ? l * 0.f : ex2((m - top) * scale_log2);
}

// The workspace: who has cut what, which CTAs had units, then the partial results.  A Cut belongs to a (sequence,
// key head, pass) where the call has fewer of those than CTAs, else to the CTA that begins it, so that decode_join_kernel
// looks at few of them.  CTA c has two places for partial results, 2 c for the part that continues what the CTA before began
// and 2 c + 1 for the one that it begins; a place is m, l of `rows` rows and their o.
struct Cut {
  int b, h;         // as in Walk
  int first, last;  // stretches that have its first and its last unit; last below 0: it is not cut
};
struct Workspace {
  int4* cuts;
  int* counts;  // of each CTA: whether it has any units
  float* parts;
  __host__ __device__ static long long floats(long long slots, long long ctas, int rows, int D) {
    return 4 * slots + (ctas + 3) / 4 * 4 + 2 * ctas * rows * (D + 2);
  }
  __device__ Workspace(float* p, int slots, int ctas)
      : cuts(reinterpret_cast<int4*>(p)), counts(reinterpret_cast<int*>(p + 4 * slots)), parts(p + 4 * slots + (ctas + 3) / 4 * 4) {}
  __device__ float* part(int place, int rows, int D) const { return parts + static_cast<long long>(place) * rows * (D + 2); }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on `bar` once the copies that this thread has started have come in.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// TILED: keys and values come in tiled copies of `box_rows` rows; else (one row) 16 bytes a lane.
template <int DP, int HP, int NT, bool BF16, bool TILED>
__global__ void __launch_bounds__(32 * kWarps, DecodeCfg<DP, HP>::kCtasPerSm)
    decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ DecodeArgs a, int rows, int slots, int box_rows, int* status) {
  using C = DecodeCfg<DP, HP>;
  constexpr int kRows = 8 * NT, kSteps = DP / 16;  // columns of a head in sixteens
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem);
  if (base & 1023u) {  // swizzled tiles need 1024-byte alignment
    if (threadIdx.x == 0) atomicCAS(status, 0, 0x20000 | kSiteDecode);
    return;
  }
  const uint32_t ring = base + warp * C::kWarpBytes;
  float* const join = reinterpret_cast<float*>(smem + C::kOffJoin);   // [kWarps][kJoinRows][kJoinStride]
  float* const join_ml = join + kWarps * kJoinRows * C::kJoinStride;  // [kWarps][kJoinRows][2]
  auto bar = [&](int stage) { return base + C::kOffBar + 8u * (warp * C::kStages + stage); };
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffAbort);
  const WaitCtx w{abort_flag, status};
  const int group = a.Hq / a.Hkv, blocks = (group + kRows - 1) / kRows;
  const int stretches = gridDim.x / blocks, stretch = blockIdx.x / blocks, pass = blockIdx.x - stretch * blocks;
  const int heads = a.Hkv / HP, d8 = a.D / 8;

  if (lane == 0)
    for (int s = 0; s < C::kStages; ++s) mbar_init(bar(s), TILED ? 1 : 32);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    if constexpr (TILED) {
      prefetch_tensormap(&tk);
      prefetch_tensormap(&tv);
    }
  }
  if constexpr (!TILED)  // columns beyond the head dim, which no copy touches
    for (int i = lane; i < C::kWarpBytes / 16; i += 32)
      *reinterpret_cast<uint4*>(smem + warp * C::kWarpBytes + i * 16) = make_uint4(0, 0, 0, 0);
  fence_mbar_init();
  fence_proxy_async_smem();
  __syncthreads();
  grid_wait_previous();
  grid_allow_next();

  const Workspace space(a.workspace, slots, gridDim.x);
  const bool by_segment = static_cast<long long>(a.batch) * heads * blocks == slots;  // what a Cut belongs to
  // sequences without keys, and those with more than the block table has room for (2^31 - 1: as many as that)
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const int n = ld_global(a.lengths + b);
    if (threadIdx.x == 0 && n != 0x7fffffff && n > static_cast<long long>(a.table_width) * a.page_size)
      atomicCAS(status, 0, kStatusPage | kSiteDecode);
    if (n <= 0) {
      for (int i = threadIdx.x; i < a.Hq * d8; i += 32 * kWarps)
        reinterpret_cast<uint4*>(a.out)[static_cast<long long>(b) * a.Hq * d8 + i] = make_uint4(0, 0, 0, 0);
      if (by_segment)
        for (int h = threadIdx.x; h < heads * blocks; h += 32 * kWarps) space.cuts[b * heads * blocks + h] = make_int4(0, 0, 0, -1);
    }
  }

  const long long total = row_length(a, heads, lane);
  const long long u0 = stretch_start(total, stretch, stretches), u1 = stretch_start(total, stretch + 1, stretches);
  Walk load{0, 0, 0, 0, 0, static_cast<int>(u1 - u0)};
  if (load.left > 0) find_unit(a, heads, u0, lane, load);
  if (threadIdx.x == 0) space.counts[blockIdx.x] = load.left > 0;
  if (load.left <= 0) {
    if (!by_segment && threadIdx.x == 0) space.cuts[blockIdx.x] = make_int4(0, 0, 0, -1);
    return;
  }
  Walk work = load;

  // ---- loading: unit n of the stretch into stage n % kStages; lane i looks after box i of the warp's 16 keys.  The page
  // number of the next unit's box is on its way while this one is waited for and worked on.
  const int boxes = 16 / box_rows;
  int page = -1, slot = 0;
  auto look_up = [&]() {
    const int key = load.unit * kUnit + warp * 16 + lane * box_rows;
    page = -1;
    if (lane < boxes && key < load.length) {
      const int index = key / a.page_size;
      slot = key - index * a.page_size;
      page = ld_global(a.block_table + load.b * a.table_stride + index);
    }
  };
  auto issue = [&](int stage) {
    const int key = load.unit * kUnit + warp * 16 + lane * box_rows;
    const bool asked = lane < boxes && key < load.length;
    const bool take = asked && page >= 0 && page < a.pages;
    if (asked && !take) atomicCAS(status, 0, kStatusPage | kSiteDecode);
    const int copies = __popc(__ballot_sync(0xffffffffu, take));
    // keys of this lane's box that count
    const int here = take ? min(load.length - key, box_rows) : 0;
    uint32_t keys = here > 0 ? ((1u << here) - 1u) << (lane * box_rows) : 0u;
    keys = __reduce_or_sync(0xffffffffu, keys);
    if (copies != 0) {
      const uint32_t dst = ring + stage * 2 * C::kTileBytes;
      if constexpr (TILED) {
        if (lane == 0) mbar_arrive_expect_tx(bar(stage), copies * box_rows * C::kWide * 4);
        __syncwarp();
        if (take) {
#pragma unroll
          for (int ch = 0; ch < C::kChunks; ++ch) {
            const uint32_t to = dst + ch * 2048 + lane * box_rows * 128;
            const int x = HP == 2 ? 0 : ch * 64;
            const HeadCoord from{HP == 2 ? 2 * load.h + ch : load.h, page};
            tma_load_4d(to, &tk, x, slot, from, bar(stage));
            tma_load_4d(to + C::kTileBytes, &tv, x, slot, from, bar(stage));
          }
        }
      } else {
        // lane i has piece i % kPieces of every (32 / kPieces)-th row; columns beyond the head dim stay the zeros that they are
        constexpr int kPieces = C::kWide / 8;
        const int piece = lane % kPieces, chunk = piece / 8, column = HP == 2 ? piece % 8 : piece;
        const long long kh = (HP == 2 ? 2 * load.h + chunk : load.h) * a.sk_cache.head + column * 8;
        const long long vh = (HP == 2 ? 2 * load.h + chunk : load.h) * a.sv_cache.head + column * 8;
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += 32 / kPieces) {
          const int row = r0 + lane / kPieces, p = __shfl_sync(0xffffffffu, take ? page : -1, row);
          const long long at = __shfl_sync(0xffffffffu, slot, row);
          if (p >= 0 && column < d8) {
            const uint32_t to = dst + chunk * 2048 + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
            copy16(to, static_cast<const uint16_t*>(a.k_cache) + p * a.sk_cache.page + at * a.sk_cache.slot + kh);
            copy16(to + C::kTileBytes, static_cast<const uint16_t*>(a.v_cache) + p * a.sv_cache.page + at * a.sv_cache.slot + vh);
          }
        }
        copies_arrive(bar(stage));
      }
    }
    next_unit(a, heads, load);
    if (load.left > 0) look_up();
    return keys;
  };
  look_up();
  uint32_t valid[C::kStages];  // which of its 16 keys the stage of unit n, n + 1, .. holds
#pragma unroll
  for (int s = 0; s < C::kStages; ++s) valid[s] = load.left > 0 ? issue(s) : 0u;

  uint32_t qb[HP][kSteps][NT][2];
  float o[HP][kSteps][NT][4];  // rows (columns of V) 16 i + lane / 4 (+ 8), columns (query heads) 8 t + 2 (lane % 4) (+ 1)
  float m[HP][NT][2], l[HP][NT][2];
  // (finite for any scale, so that a first finite score is above it)
  const float threshold = fminf(weight_lag<BF16>(8.f) / a.scale_log2, 3e38f);
  uint32_t phases = 0;  // bit s: parity of the next wait on stage s
  bool fresh = true, ok = true;
  bool begins = work.unit == 0;  // the first unit of the (sequence, key head) is in this stretch
  int stage = 0;
  const int here = min(kRows, group - pass * kRows);  // query heads in use
  auto load_q = [&]() {
#pragma unroll
    for (int p = 0; p < HP; ++p) {
      const uint16_t* const q =
          static_cast<const uint16_t*>(a.q) + work.b * a.sq.row + ((work.h * HP + p) * group + pass * kRows) * a.sq.head;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int head = 8 * t + lane / 4, col = 16 * i + 8 * j + (lane & 3) * 2;
            qb[p][i][t][j] = head < here && col < a.D ? ld_global(reinterpret_cast<const unsigned*>(q + head * a.sq.head + col)) : 0u;
          }
    }
  };
  load_q();
  while (work.left > 0) {
    if (fresh) {
#pragma unroll
      for (int p = 0; p < HP; ++p)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          m[p][t][0] = m[p][t][1] = -INFINITY;
          l[p][t][0] = l[p][t][1] = 0.f;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) o[p][i][t][0] = o[p][i][t][1] = o[p][i][t][2] = o[p][i][t][3] = 0.f;
        }
    }
    // ---- one unit: this warp's 16 keys
    const uint32_t mine = valid[0];
    if (mine != 0) {
      if (ok) ok = mbar_wait_warp(bar(stage), (phases >> stage) & 1u, w, kSiteDecode);
      phases ^= 1u << stage;
      const uint32_t ktile = ring + stage * 2 * C::kTileBytes, vtile = ktile + C::kTileBytes;
      if (mine != 0xffffu) {  // rows that do not count: 0 x NaN is none
        for (int i = lane; i < 16 * C::kChunks * 8; i += 32)
          if (!((mine >> (i / 8 % 16)) & 1u))
            *reinterpret_cast<uint4*>(smem + (vtile - base) + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      // row of this lane in the 16 x 16 piece of a tile that ldmatrix takes, and which half of its columns
      const int krow = (lane & 7) + (lane & 8), khalf = lane >> 4;
      const bool in0 = (mine >> (lane / 4)) & 1u, in1 = (mine >> (lane / 4 + 8)) & 1u;
      float s[HP][NT][4] = {};
      bool need = false;
#pragma unroll
      for (int p = 0; p < HP; ++p) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t x[4];
          load_matrices(ktile + ((p * kSteps + k) / 4) * 2048 + krow * 128 + (((2 * (k % 4) + khalf) ^ (krow & 7)) << 4), x);
#pragma unroll
          for (int t = 0; t < NT; ++t) product<BF16>(s[p][t], x, qb[p][k][t][0], qb[p][k][t][1]);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (!in0) s[p][t][e] = -INFINITY;
            if (!in1) s[p][t][2 + e] = -INFINITY;
            need |= fmaxf(s[p][t][e], s[p][t][2 + e]) - m[p][t][e] > threshold;
          }
      }
      // The maximum follows only when a score is 2^8 (fp16: 2^4) above it: a weight is at most 2^8 (P 2^11 at fp16: 2^15) then.
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int p = 0; p < HP; ++p)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = fmaxf(s[p][t][e], s[p][t][2 + e]);
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              x = fmaxf(x, m[p][t][e]);
              // a head without a finite score so far has weights 0
              const float alpha = x == -INFINITY ? 1.f : ex2((m[p][t][e] - x) * a.scale_log2);
              m[p][t][e] = x;
              l[p][t][e] *= alpha;
#pragma unroll
              for (int i = 0; i < kSteps; ++i) o[p][i][t][e] *= alpha, o[p][i][t][2 + e] *= alpha;
            }
      }
      // P^T in 16 bits, with kWeightPower, which cancels in the end; at bf16, whose 8 bits would be the largest error of the output, as a sum of two.  The first
      // term is p (1 - 2^-8) rounded, at most p (1 - 2^-16), so that the second one is positive where p is, and an
      // infinite value stays infinite in both products.  At fp16 one term's 11 bits are those of the output: its error is 1.34 times
      // that of its rounding alone (2.78e-4 against 2.08e-4 of its norm, 32 sequences of 100 to 2000, 12 heads of 64), and a second term took
      // 20.1 -> 21.05 us there, 125.6 -> 133 on 64 of 500 to 8192, 32 / 2 heads of 256, 83.2 -> 90.7 on 64 / 2 of 128.
      // V^T: the 16 x 16 piece of V is turned around on its way, so the lanes' rows and halves change places.
      const int vrow = (lane & 7) + ((lane >> 4) << 3), vhalf = (lane >> 3) & 1;
#pragma unroll
      for (int p = 0; p < HP; ++p) {
        uint32_t weight[NT][2], rest[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float shift = m[p][t][e] == -INFINITY ? 0.f : kWeightPower<BF16> - m[p][t][e] * a.scale_log2;
            s[p][t][e] = ex2(fmaf(s[p][t][e], a.scale_log2, shift));
            s[p][t][2 + e] = ex2(fmaf(s[p][t][2 + e], a.scale_log2, shift));
            l[p][t][e] += s[p][t][e] + s[p][t][2 + e];
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = s[p][t][2 * j], y = s[p][t][2 * j + 1];
            if constexpr (BF16) {
              const uint32_t both = pack2<BF16>(x * 0.99609375f, y * 0.99609375f);
              const float2 f = unpack2<BF16>(both);
              weight[t][j] = turned(both);
              rest[t][j] = turned(pack2<BF16>(x - f.x, y - f.y));
            } else {
              weight[t][j] = turned(pack2<BF16>(x, y));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t x[4];
          load_matrices_t(vtile + ((p * kSteps + i) / 4) * 2048 + vrow * 128 + (((2 * (i % 4) + vhalf) ^ (vrow & 7)) << 4), x);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            product<BF16>(o[p][i][t], x, weight[t][0], weight[t][1]);
            if constexpr (BF16) product<BF16>(o[p][i][t], x, rest[t][0], rest[t][1]);
          }
        }
      }
    }
    __syncwarp();
    // ---- the next load takes the stage of this unit
#pragma unroll
    for (int s = 0; s + 1 < C::kStages; ++s) valid[s] = valid[s + 1];
    valid[C::kStages - 1] = ok && load.left > 0 ? issue(stage) : 0u;
    if (++stage == C::kStages) stage = 0;

    // ---- the end of a (sequence, key head), or of the stretch: the warps' sums become one, eight heads at a time, with the
    // next queries on their way
    const Walk now = work;
    const bool ends = now.unit + 1 == now.units;
    next_unit(a, heads, work);
    fresh = ends || work.left <= 0;
    if (fresh) {
      if (work.left > 0) load_q();
      const bool whole = begins && ends;
      float* const part = space.part(2 * blockIdx.x + (begins ? 1 : 0), HP * rows, a.D);
      if (threadIdx.x == 0 && (by_segment ? begins : work.left <= 0)) {
        // the stretch of a unit is the last one that starts at or before it
        const long long last = u1 - now.left + (now.units - 1 - now.unit);
        const int end = begins && !ends ? static_cast<int>(((last + 1) * stretches - 1) / total) : -1;
        space.cuts[by_segment ? (now.b * heads + now.h) * blocks + pass : blockIdx.x] = make_int4(now.b, now.h, stretch, end);
      }
      begins = true;
#pragma unroll
      for (int pt = 0; pt < HP * NT; ++pt) {
        const int p = pt / NT, t = pt % NT;
        const int row0 = t * kJoinRows, some = min(here - row0, kJoinRows);
        if (some <= 0) continue;
        const int head0 = (now.h * HP + p) * group + pass * kRows + row0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[p][t][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int row = warp * kJoinRows + (lane & 3) * 2 + e;
          float* const to = join + row * C::kJoinStride + lane / 4;
#pragma unroll
          for (int i = 0; i < kSteps; ++i) to[16 * i] = o[p][i][t][e], to[16 * i + 8] = o[p][i][t][2 + e];
          if (lane < 4) *reinterpret_cast<float2*>(join_ml + row * 2) = make_float2(m[p][t][e], sum);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < some * (a.D / 2); i += 32 * kWarps) {
          const int row = i / (a.D / 2), col = (i - row * (a.D / 2)) * 2;
          float mw[kWarps], top = -INFINITY;
#pragma unroll
          for (int v = 0; v < kWarps; ++v) top = fmaxf(top, mw[v] = join_ml[(v * kJoinRows + row) * 2]);
          float2 sum = make_float2(0.f, 0.f);
          float all = 0.f;
#pragma unroll
          for (int v = 0; v < kWarps; ++v) {
            const float lw = join_ml[(v * kJoinRows + row) * 2 + 1];
            const float f = part_weight(mw[v], lw, top, a.scale_log2);
            const float2 x = *reinterpret_cast<const float2*>(join + (v * kJoinRows + row) * C::kJoinStride + col);
            sum.x = fmaf(f, x.x, sum.x);
            sum.y = fmaf(f, x.y, sum.y);
            all = fmaf(f, lw, all);
          }
          if (whole) {
            const float inv = 1.f / all;
            uint16_t* const to = static_cast<uint16_t*>(a.out) + (static_cast<long long>(now.b) * a.Hq + head0 + row) * a.D + col;
            *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(sum.x * inv, sum.y * inv);
          } else {
            const int r = p * rows + row0 + row;  // of the place
            *reinterpret_cast<float2*>(part + 2 * HP * rows + r * a.D + col) = sum;
            if (col == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(top, all);
          }
        }
        __syncthreads();
      }
    }
  }
}

// Adds up the parts of what decode_kernel's stretches cut apart: block (c, row) one query head of Cut c.  Shares of D / 2 threads
// take every n-th part, several at a time with their maxima and sums, so that a share waits for memory once for
// kJoinBatch parts; then the shares become one.  Few long sequences have a hundred parts and more to a head: one thread a
// column, part after part, took 73 us on two sequences of 131 072 keys, weights first and the parts behind them 13.5.
constexpr int kJoinMost = 512, kJoinBatch = 8;
template <bool BF16>
__global__ void __launch_bounds__(kJoinMost) decode_join_kernel(const __grid_constant__ DecodeArgs a, int rows, int pass_heads, int hp,
                                                                int slots, int ctas) {
  __shared__ float4 shared[kJoinMost];  // sums of two columns, maximum, sum of the weights
  grid_wait_previous();
  // No grid_allow_next: CTAs of the next decode_kernel that start under this one find its small blocks of shared memory taken in the middle
  // of an SM's and settle around them; what these leave behind is in two pieces, too small for the SM's last CTA, which then
  // runs after the others (64 sequences of 204 000 keys, 12 heads of 64 columns: 170 us against 134).  So it starts when the last CTA
  // here has ended, which is 2 us earlier than an ordinary launch (two of 131 072 keys: 56 -> 53.5, 345 000 keys in 128: 237 -> 233).
  const Workspace space(a.workspace, slots, ctas);
  const int place_rows = hp * rows, row = blockIdx.x % place_rows;
  const uint4 c = ld_global(reinterpret_cast<const uint4*>(space.cuts) + blockIdx.x / place_rows);
  const Cut cut{static_cast<int>(c.x), static_cast<int>(c.y), static_cast<int>(c.z), static_cast<int>(c.w)};
  const int group = a.Hq / a.Hkv, blocks = (group + pass_heads - 1) / pass_heads, pass = blockIdx.x / place_rows % blocks;
  const int in_group = pass * pass_heads + row % rows;
  if (cut.last < 0 || in_group >= group) return;
  const int parts = cut.last - cut.first + 1, d2 = a.D / 2;
  const int col = threadIdx.x % d2, share = threadIdx.x / d2, shares = blockDim.x / d2;
  float top = -INFINITY, all = 0.f;
  float2 sum = make_float2(0.f, 0.f);
  auto add = [&](float m, float l, float2 x, float now) {
    const float f = part_weight(m, l, now, a.scale_log2);
    all = fmaf(f, l, all);
    sum.x = fmaf(f, x.x, sum.x);  // (0 x NaN is NaN in whichever part it stands)
    sum.y = fmaf(f, x.y, sum.y);
  };
  auto lower = [&](float now) {
    const float old = part_weight(top, all, now, a.scale_log2);
    all *= old, sum.x *= old, sum.y *= old;
    top = now;
  };
  if (share < shares)
    for (int i0 = share; i0 < parts; i0 += kJoinBatch * shares) {
      float2 ml[kJoinBatch], x[kJoinBatch];
      int some[kJoinBatch];
#pragma unroll
      for (int j = 0; j < kJoinBatch; ++j) {
        const int i = min(i0 + j * shares, parts - 1), cta = (cut.first + i) * blocks + pass;
        const float* const at = space.part(2 * cta + (i == 0 ? 1 : 0), place_rows, a.D);
        // a CTA without units (there are fewer units than CTAs) has left nothing
        some[j] = i0 + j * shares < parts ? ld_global(space.counts + cta) : 0;
        ml[j] = ld_global(reinterpret_cast<const float2*>(at + 2 * row));
        x[j] = ld_global(reinterpret_cast<const float2*>(at + 2 * place_rows + row * a.D + 2 * col));
      }
      float now = top;
#pragma unroll
      for (int j = 0; j < kJoinBatch; ++j) {
        if (!some[j]) ml[j] = make_float2(-INFINITY, 0.f), x[j] = make_float2(0.f, 0.f);  // the place may hold anything
        now = fmaxf(now, ml[j].x);
      }
      lower(now);
#pragma unroll
      for (int j = 0; j < kJoinBatch; ++j) add(ml[j].x, ml[j].y, x[j], now);
    }
  shared[threadIdx.x] = make_float4(sum.x, sum.y, top, all);
  __syncthreads();
  if (share == 0) {
    for (int i = 1; i < shares; ++i) {
      const float4 x = shared[i * d2 + col];
      const float now = fmaxf(top, x.z);
      lower(now);
      add(x.z, x.w, make_float2(x.x, x.y), now);
    }
    const float inv = 1.f / all;  // NaN for a row without any finite score, as everywhere
    uint16_t* const to = static_cast<uint16_t*>(a.out) + (static_cast<long long>(cut.b) * a.Hq + (cut.h * hp + row / rows) * group + in_group) * a.D + 2 * col;
    *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(sum.x * inv, sum.y * inv);
  }
}

// CTAs of decode_kernel, of `slots` that run at a time: a multiple of the passes, no more than units of the call.
struct DecodeGrid {
  int hp, rows, ctas, cuts;  // key heads and query heads that a pass takes; CTAs; Cuts
};
DecodeGrid decode_grid(int batch, int Hq, int Hkv, int D, int table_width, int page_size, int slots) {
  const int hp = heads_at_once(Hkv, D), group = Hq / Hkv, take = 8 * column_tiles(group), passes = (group + take - 1) / take;
  const long long units = (static_cast<long long>(table_width) * page_size + kUnit - 1) / kUnit * batch * (Hkv / hp);
  const long long stretches = std::max(1, slots / passes), segments = static_cast<long long>(batch) * (Hkv / hp) * passes;
  const int ctas = static_cast<int>(std::min(units, stretches) * passes);
  return DecodeGrid{hp, std::min(group, take), ctas, static_cast<int>(std::min<long long>(segments, ctas))};
}

template <int DP, int HP, int NT, bool BF16, bool TILED>
cudaError_t launch_decode_s(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeArgs& a, int box_rows, int num_sms, int* status,
                            cudaStream_t stream) {
  using C = DecodeCfg<DP, HP>;
  auto kern = decode_kernel<DP, HP, NT, BF16, TILED>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return e;
  const DecodeGrid g = decode_grid(a.batch, a.Hq, a.Hkv, a.D, a.table_width, a.page_size, std::min(num_sms * C::kCtasPerSm, kMaxCtas));
  e = launch_dependent(kern, g.ctas, 32 * kWarps, C::kSmemBytes, stream, tk, tv, a, g.rows, g.cuts, box_rows, status);
  if (e != cudaSuccess) return e;
  // as many shares as take the parts of a cut at once, were the cuts alike
  const int batches = (g.ctas / g.cuts + kJoinBatch) / kJoinBatch;
  const int threads = std::min(std::max(256, (a.D / 2 * batches + 31) / 32 * 32), kJoinMost);
  return launch_dependent(decode_join_kernel<BF16>, static_cast<unsigned>(g.cuts) * g.rows * HP, threads, 0, stream, a, g.rows, 8 * NT, HP, g.cuts, g.ctas);
}

// With one row to a box the tiled copies themselves bound the kernel.  64 sequences of 204 000 keys, 32 / 8 heads of 128 columns,
// microseconds with tiled copies / 16 bytes a lane, pages of 1: 309 / 219, 2: 216 / 217, 4: 164 / 212, 8: 148 / 211; of
// 131 000 keys, 16 / 2 heads of 256 columns, pages of 1: 171 / 106, 2: 116 / 107, 4: 84 / 105.
template <int DP, int HP, int NT, bool BF16>
cudaError_t launch_decode_t(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeArgs& a, int box_rows, int num_sms, int* status,
                            cudaStream_t stream) {
  return box_rows > 1 ? launch_decode_s<DP, HP, NT, BF16, true>(tk, tv, a, box_rows, num_sms, status, stream)
                      : launch_decode_s<DP, HP, NT, BF16, false>(tk, tv, a, box_rows, num_sms, status, stream);
}

}  // namespace

size_t decode_workspace_floats(int batch, int Hq, int Hkv, int D, int table_width, int page_size) {
  // (more CTAs than this never run; the largest number of passes may need more)
  const DecodeGrid g = decode_grid(batch, Hq, Hkv, D, table_width, page_size, kMaxCtas);
  return static_cast<size_t>(Workspace::floats(g.cuts, g.ctas, g.hp * g.rows, D));
}

int decode_box_rows(int page_size) {
  int rows = 16;
  while (page_size % rows) rows /= 2;
  return rows;
}

cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeArgs& a, int dtype, int num_sms, int* status,
                          cudaStream_t stream) {
  const int box = decode_box_rows(a.page_size), tiles = column_tiles(a.Hq / a.Hkv);
#define FA2_CASE(DP, HP)                                                                                     \
  if (tiles == 1)                                                                                            \
    return dtype ? launch_decode_t<DP, HP, 1, true>(tk, tv, a, box, num_sms, status, stream)                 \
                 : launch_decode_t<DP, HP, 1, false>(tk, tv, a, box, num_sms, status, stream);               \
  return dtype ? launch_decode_t<DP, HP, 2, true>(tk, tv, a, box, num_sms, status, stream)                   \
               : launch_decode_t<DP, HP, 2, false>(tk, tv, a, box, num_sms, status, stream)
  if (a.D <= 64 && heads_at_once(a.Hkv, a.D) == 2) { FA2_CASE(64, 2); }
  if (a.D <= 64) { FA2_CASE(64, 1); }
  if (a.D <= 128) { FA2_CASE(128, 1); }
  FA2_CASE(256, 1);
#undef FA2_CASE
}

}  // namespace fa2
