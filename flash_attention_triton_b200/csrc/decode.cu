// Attention of one new token a sequence over its pages of a key-value cache.
//
//     out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),  j < lengths[b]
//
// Bound by reading the keys and values once.  The keys of every (sequence, key head) are cut into units of 64; all
// units of the call stand in one row, and each CTA takes an equal stretch of it, whatever the lengths are, so
// one long sequence and many short ones both keep every SM reading.  Where a stretch cuts a (sequence, key head)
// apart, each CTA leaves (m, l, o) of its part in the workspace, and decode_join_kernel adds the parts up in order:
// the same bits every time.
//
// Inside a CTA warp w takes keys 16 w .. 16 w + 15 of every unit and runs on its own: its keys and values arrive
// by 16-byte asynchronous copies in a ring of stages of its own, the query heads of the key head are the rows of
// m16n8k16 products (S = Q K^T, O += P V, fp32 accumulators in registers), and maximum and sum of the softmax
// run along.  The four warps meet where a (sequence, key head) ends, while their next stages are already loading.
// The products cost a fifth of the time that the bytes take, so the mma.sync form does, and a row of
// 16 queries needs no tile of 128.
#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace fa2 {
namespace {

constexpr int kUnit = 64;  // keys
constexpr int kWarps = 4;
constexpr int kRows = 16;  // query heads of a key head that one pass takes
constexpr int kJoinRows = 8;  // rows that the warps of a CTA add up at a time
constexpr int kMaxCtas = 1024;

template <int DP>
struct DecodeCfg {
  static constexpr int kStages = DP == 64 ? 4 : 3;
  static constexpr int kCtasPerSm = DP == 64 ? 3 : (DP == 128 ? 2 : 1);
  static constexpr int kTileBytes = 16 * DP * 2;                           // 16 keys, or 16 values
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kJoinStride = DP + 4;                               // floats of a row of partial sums
  static constexpr int kSmemBytes = kWarps * kWarpBytes + kWarps * kJoinRows * (kJoinStride + 2) * 4;
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory of one SM");
};

// One (sequence, row of heads) of the call, and the walk over the units of a CTA's stretch.
struct Walk {
  int b, h;        // sequence; key head and, where it has more than 16 query heads, which 16 of them
  int unit;        // next unit of it
  int units;       // units of the sequence
  int length;      // keys of the sequence
};

__device__ __forceinline__ int clamp_length(const DecodeArgs& a, int b) {
  const long long most = static_cast<long long>(a.table_width) * a.page_size;
  const long long n = ld_global(a.lengths + b);
  return static_cast<int>(n < 0 ? 0 : (n > most ? most : n));
}
__device__ __forceinline__ int units_of(int length) { return (length + kUnit - 1) / kUnit; }

// Units of all sequences, and of those before sequence `b` (whole warp).
__device__ __forceinline__ long long units_before(const DecodeArgs& a, int b, int lane) {
  long long sum = 0;
  for (int i = 0; i < b; i += 32) {
    const unsigned u = i + lane < b ? units_of(clamp_length(a, i + lane)) : 0;
    sum += __reduce_add_sync(0xffffffffu, u);
  }
  return sum;
}

__device__ __forceinline__ long long stretch_start(long long total, int cta, int ctas) { return total * cta / ctas; }

// Puts `w` on unit `at` of the row (whole warp); the row has more than `at` units.
__device__ __forceinline__ void find_unit(const DecodeArgs& a, int heads, long long at, int lane, Walk& w) {
  for (int i = 0;; i += 32) {
    const int n = i + lane < a.batch ? clamp_length(a, i + lane) : 0;
    const unsigned mine = units_of(n);
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
    w.b = i + l;
    w.units = __shfl_sync(0xffffffffu, mine, l);
    w.length = __shfl_sync(0xffffffffu, n, l);
    const int rest = static_cast<int>(at - static_cast<long long>(__shfl_sync(0xffffffffu, upto - mine, l)) * heads);
    w.h = rest / w.units;
    w.unit = rest - w.h * w.units;
    return;
  }
}

// To the next unit of the row; there is one.
__device__ __forceinline__ void next_unit(const DecodeArgs& a, int heads, Walk& w) {
  if (++w.unit < w.units) return;
  w.unit = 0;
  if (++w.h < heads) return;
  w.h = 0;
  do {
    w.length = ++w.b < a.batch ? clamp_length(a, w.b) : 1;
    w.units = units_of(w.length);
  } while (w.units == 0);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
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

// The workspace: for each CTA what it has begun and not ended, then the partial results.  CTA c has two places for those,
// 2 c for the part that continues what the CTA before began and 2 c + 1 for the one that it begins; a place is m, l of
// `rows` rows and their o.
struct Cut {
  int b, h;  // as in Walk
  int last;  // CTA that has the last unit; below 0: it has ended what it began
  int units; // of the CTA's stretch
};
__device__ __forceinline__ float* partial(float* workspace, int ctas, int place, int rows, int D) {
  return workspace + ctas * 4 + static_cast<long long>(place) * rows * (D + 2);
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(32 * kWarps, DecodeCfg<DP>::kCtasPerSm)
    decode_kernel(const __grid_constant__ DecodeArgs a, int rows, int* status) {
  using C = DecodeCfg<DP>;
  constexpr int kPieces = DP / 8;  // 16-byte pieces of a row
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + warp * C::kWarpBytes;
  float* const join = reinterpret_cast<float*>(smem + kWarps * C::kWarpBytes);  // [kWarps][kJoinRows][kJoinStride]
  float* const join_ml = join + kWarps * kJoinRows * C::kJoinStride;            // [kWarps][kJoinRows][2]
  const int group = a.Hq / a.Hkv, blocks = (group + kRows - 1) / kRows;
  const int heads = a.Hkv * blocks;
  const int d8 = a.D / 8;

  // columns beyond the head dim are zeros that no copy touches
  if (d8 < kPieces)
    for (int i = lane; i < C::kWarpBytes / 16; i += 32)
      *reinterpret_cast<uint4*>(smem + warp * C::kWarpBytes + i * 16) = make_uint4(0, 0, 0, 0);
  __syncwarp();
  grid_wait_previous();
  grid_allow_next();

  // sequences without keys
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
    if (ld_global(a.lengths + b) <= 0)
      for (int i = threadIdx.x; i < a.Hq * d8; i += 32 * kWarps)
        reinterpret_cast<uint4*>(a.out)[static_cast<long long>(b) * a.Hq * d8 + i] = make_uint4(0, 0, 0, 0);

  const long long total = units_before(a, a.batch, lane) * heads;
  const long long u0 = stretch_start(total, blockIdx.x, gridDim.x);
  const int count = static_cast<int>(stretch_start(total, blockIdx.x + 1, gridDim.x) - u0);
  Cut* const cut = reinterpret_cast<Cut*>(a.workspace) + blockIdx.x;
  if (count == 0) {
    if (threadIdx.x == 0) *reinterpret_cast<int4*>(cut) = make_int4(0, 0, -1, 0);
    return;
  }
  Walk load;
  find_unit(a, heads, u0, lane, load);
  Walk work = load;

  // ---- loading: unit n of the stretch into stage n % kStages; lane i looks after key i % 16 of the warp's 16
  auto issue = [&](int stage) {
    const int key = load.unit * kUnit + warp * 16 + (lane & 15);
    int page = -1, slot = 0;
    if (key < load.length) {
      const int index = key / a.page_size;
      slot = key - index * a.page_size;
      page = ld_global(a.block_table + load.b * a.table_stride + index);
      if (page < 0 || page >= a.pages) {
        atomicCAS(status, 0, kStatusPage | kSiteDecode);
        page = -1;
      }
    }
    const uint32_t here = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
    if (here != 0) {
      const int kv_head = load.h / blocks;
      const uint16_t* const kbase = static_cast<const uint16_t*>(a.k_cache) + kv_head * a.sk_cache.head;
      const uint16_t* const vbase = static_cast<const uint16_t*>(a.v_cache) + kv_head * a.sv_cache.head;
      const uint32_t dst = ring + stage * 2 * C::kTileBytes;
#pragma unroll
      for (int i = 0; i < 16 * kPieces / 32; ++i) {
        const int row = (lane + 32 * i) / kPieces, piece = (lane + 32 * i) % kPieces;
        const int p = __shfl_sync(0xffffffffu, page, row), s = __shfl_sync(0xffffffffu, slot, row);
        if (piece < d8) {
          const uint32_t to = dst + row * (DP * 2) + ((piece ^ (row & 7)) << 4);
          const bool take = p >= 0;  // zeros otherwise: their weight is zero, and 0 x NaN is none
          const long long pp = take ? p : 0, sl = take ? s : 0;
          copy16(to, kbase + pp * a.sk_cache.page + sl * a.sk_cache.slot + piece * 8, take);
          copy16(to + C::kTileBytes, vbase + pp * a.sv_cache.page + sl * a.sv_cache.slot + piece * 8, take);
        }
      }
    }
    return here;
  };
  uint32_t valid[C::kStages];  // which of its 16 keys the stage of unit n, n + 1, .. holds
  int issued = 0;
#pragma unroll
  for (int s = 0; s < C::kStages; ++s) {
    valid[s] = 0;
    if (issued < count) {
      valid[s] = issue(s);
      if (++issued < count) next_unit(a, heads, load);
    }
    copies_commit();
  }

  uint32_t qa[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  bool fresh = true;
  for (int n = 0; n < count; ++n) {
    const int head0 = work.h / blocks * group + work.h % blocks * kRows;    // first query head of the rows
    const int here = min(kRows, group - work.h % blocks * kRows);           // rows in use
    if (fresh) {
      fresh = false;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      const uint16_t* const q = static_cast<const uint16_t*>(a.q) + work.b * a.sq.row;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = lane / 4 + (i & 1) * 8, col = k * 16 + (lane & 3) * 2 + (i >> 1) * 8;
          qa[k][i] = row < here && col < a.D
                         ? ld_global(reinterpret_cast<const unsigned*>(q + (head0 + row) * a.sq.head + col)) : 0u;
        }
    }
    // ---- one unit: this warp's 16 keys
    copies_wait<C::kStages - 1>();
    __syncwarp();
    const uint32_t mine = valid[0];
    if (mine != 0) {
      const uint32_t ktile = ring + (n % C::kStages) * 2 * C::kTileBytes, vtile = ktile + C::kTileBytes;
      const int mrow = (lane & 7) + ((lane >> 4) << 3), mpiece = (lane >> 3) & 1;  // of this lane's matrix row
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t b[4];
        load_matrices(ktile + mrow * (DP * 2) + (((2 * k + mpiece) ^ (mrow & 7)) << 4), b);
        product<BF16>(s[0], qa[k], b[0], b[1]);
        product<BF16>(s[1], qa[k], b[2], b[3]);
      }
      if (mine != 0xffffu) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((mine >> (t * 8 + (lane & 3) * 2 + (i & 1))) & 1u)) s[t][i] = -INFINITY;
      }
      float alpha[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        const float was = m[r];
        m[r] = fmaxf(was, x);
        // a row without a finite score so far has weights 0
        alpha[r] = m[r] == -INFINITY ? 1.f : ex2((was - m[r]) * a.scale_log2);
        const float base = m[r] == -INFINITY ? 0.f : -m[r] * a.scale_log2;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) sum += s[t][2 * r + e] = ex2(fmaf(s[t][2 * r + e], a.scale_log2, base));
        l[r] = l[r] * alpha[r] + sum;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][0] *= alpha[0], o[i][1] *= alpha[0];
          o[i][2] *= alpha[1], o[i][3] *= alpha[1];
        }
      }
      // P in 16 bits; at bf16, whose 8 bits would be the largest error of the output, as a sum of two.  The first
      // term is p (1 - 2^-8) rounded, at most p (1 - 2^-16), so that the second one is positive where p is, and an
      // infinite value stays infinite in both products.
      uint32_t p[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
        if constexpr (BF16) {
          p[i] = pack2<BF16>(x * 0.99609375f, y * 0.99609375f);
          const float2 f = unpack2<BF16>(p[i]);
          rest[i] = pack2<BF16>(x - f.x, y - f.y);
        } else {
          p[i] = pack2<BF16>(x, y);
        }
      }
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t b[4];
        const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3), vpiece = lane >> 4;
        load_matrices_t(vtile + vrow * (DP * 2) + (((2 * k + vpiece) ^ (vrow & 7)) << 4), b);
        product<BF16>(o[2 * k], p, b[0], b[1]);
        product<BF16>(o[2 * k + 1], p, b[2], b[3]);
        if constexpr (BF16) {
          product<BF16>(o[2 * k], rest, b[0], b[1]);
          product<BF16>(o[2 * k + 1], rest, b[2], b[3]);
        }
      }
    }
    __syncwarp();
    // ---- the next load takes the stage of this unit
#pragma unroll
    for (int s = 0; s + 1 < C::kStages; ++s) valid[s] = valid[s + 1];
    valid[C::kStages - 1] = 0;
    if (issued < count) {
      valid[C::kStages - 1] = issue(n % C::kStages);
      if (++issued < count) next_unit(a, heads, load);
    }
    copies_commit();

    // ---- the end of a (sequence, key head), or of the stretch: the warps' sums become one, eight rows at a time
    const bool ends = work.unit + 1 == work.units;
    if (ends || n + 1 == count) {
      const bool begins = work.unit <= n;  // its first unit is in this stretch
      const bool whole = begins && ends;
      float* const part = partial(a.workspace, gridDim.x, 2 * blockIdx.x + (begins ? 1 : 0), rows, a.D);
      if (n + 1 == count && threadIdx.x == 0) {
        // the CTA of a unit is the last one whose stretch starts at or before it
        const long long last = u0 + n + (work.units - 1 - work.unit);
        const int cta = begins && !ends ? static_cast<int>(((last + 1) * gridDim.x - 1) / total) : -1;
        *reinterpret_cast<int4*>(cut) = make_int4(work.b, work.h, cta, count);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (r * kJoinRows >= here) break;
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        {
          const int row = lane / 4;
          float* const to = join + (warp * kJoinRows + row) * C::kJoinStride;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i)
            *reinterpret_cast<float2*>(to + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
          if ((lane & 3) == 0)
            *reinterpret_cast<float2*>(join_ml + (warp * kJoinRows + row) * 2) = make_float2(m[r], l[r]);
        }
        __syncthreads();
        const int row0 = r * kJoinRows, some = min(here - row0, kJoinRows);
        for (int i = threadIdx.x; i < some * (a.D / 2); i += 32 * kWarps) {
          const int row = i / (a.D / 2), col = (i - row * (a.D / 2)) * 2;
          float mw[kWarps], top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, mw[w] = join_ml[(w * kJoinRows + row) * 2]);
          float2 sum = make_float2(0.f, 0.f);
          float all = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float lw = join_ml[(w * kJoinRows + row) * 2 + 1];
            const float f = part_weight(mw[w], lw, top, a.scale_log2);
            const float2 x = *reinterpret_cast<const float2*>(join + (w * kJoinRows + row) * C::kJoinStride + col);
            sum.x = fmaf(f, x.x, sum.x);
            sum.y = fmaf(f, x.y, sum.y);
            all = fmaf(f, lw, all);
          }
          if (whole) {
            const float inv = 1.f / all;
            uint16_t* const to = static_cast<uint16_t*>(a.out) + (static_cast<long long>(work.b) * a.Hq + head0 + row0 + row) * a.D + col;
            *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(sum.x * inv, sum.y * inv);
          } else {
            *reinterpret_cast<float2*>(part + 2 * rows + (row0 + row) * a.D + col) = sum;
            if (col == 0) *reinterpret_cast<float2*>(part + 2 * (row0 + row)) = make_float2(top, all);
          }
        }
        __syncthreads();
      }
      fresh = true;
    }
    if (n + 1 < count) next_unit(a, heads, work);
  }
}

// Adds up the parts of what decode_kernel's stretches cut apart: block (c, row) one query head of what CTA c began and did
// not end.  First the weights of all parts, one a thread, then the parts, D / 2 threads to each, so that no load waits for
// another.  Few long sequences have a hundred parts and more to a head: one thread a column, part after part, took
// 73 us on two sequences of 131072 keys.
constexpr int kJoinThreads = 256;
template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const __grid_constant__ DecodeArgs a, int rows, int ctas) {
  __shared__ float weight[kJoinThreads], reduced[kJoinThreads / 32];
  __shared__ float2 sums[kJoinThreads];
  grid_wait_previous();
  grid_allow_next();
  const int c0 = blockIdx.x / rows, row = blockIdx.x - c0 * rows;
  const uint4* const cuts = reinterpret_cast<const uint4*>(a.workspace);
  const uint4 cut = ld_global(cuts + c0);  // a Cut
  const int group = a.Hq / a.Hkv, blocks = (group + kRows - 1) / kRows;
  const int h = static_cast<int>(cut.y), kv_head = h / blocks, in_group = (h - kv_head * blocks) * kRows + row;
  if (static_cast<int>(cut.z) < 0 || in_group >= group) return;
  const int parts = static_cast<int>(cut.z) - c0 + 1, d2 = a.D / 2;
  const int col = threadIdx.x % d2, share = threadIdx.x / d2, shares = kJoinThreads / d2;
  auto part = [&](int i) { return partial(a.workspace, ctas, 2 * (c0 + i) + (i == 0 ? 1 : 0), rows, a.D); };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY, all = 0.f;
  float2 sum = make_float2(0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += kJoinThreads) {
    const int here = min(parts - p0, kJoinThreads);
    float m = -INFINITY, l = 0.f;
    // a CTA without units (there are fewer units than CTAs) has left nothing
    if (threadIdx.x < here && ld_global(cuts + c0 + p0 + threadIdx.x).w != 0) {
      const float* const at = part(p0 + threadIdx.x) + 2 * row;
      m = ld_global(at), l = ld_global(at + 1);
    }
    float most = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) reduced[warp] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) most = fmaxf(most, reduced[i]);
    most = fmaxf(most, top);
    const float old = part_weight(top, all, most, a.scale_log2);
    all *= old, sum.x *= old, sum.y *= old;
    top = most;
    const float w = part_weight(m, l, top, a.scale_log2);
    weight[threadIdx.x] = w;
    l *= w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncthreads();
    if (lane == 0) reduced[warp] = l;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) all += reduced[i];
    if (share < shares)
#pragma unroll 4
      for (int i = share; i < here; i += shares) {
        const float f = weight[i];
        if (f == 0.f) continue;
        const float* const x = part(p0 + i) + 2 * rows + row * a.D + 2 * col;
        sum.x = fmaf(f, ld_global(x), sum.x);
        sum.y = fmaf(f, ld_global(x + 1), sum.y);
      }
    __syncthreads();
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (share == 0) {
    for (int i = 1; i < shares; ++i) {
      const float2 x = sums[i * d2 + col];
      sum.x += x.x, sum.y += x.y;
    }
    const float inv = 1.f / all;  // NaN for a row without any finite score, as everywhere
    uint16_t* const to = static_cast<uint16_t*>(a.out) + (static_cast<long long>(cut.x) * a.Hq + kv_head * group + in_group) * a.D + 2 * col;
    *reinterpret_cast<uint32_t*>(to) = pack2<BF16>(sum.x * inv, sum.y * inv);
  }
}

// CTAs of decode_kernel.
int decode_ctas(const DecodeArgs& a, int per_sm, int num_sms) {
  const int blocks = (a.Hq / a.Hkv + kRows - 1) / kRows;
  const long long units = (static_cast<long long>(a.table_width) * a.page_size + kUnit - 1) / kUnit;
  const long long most = units * a.batch * a.Hkv * blocks;
  const long long slots = static_cast<long long>(num_sms) * per_sm;
  return static_cast<int>(most < slots ? most : (slots < kMaxCtas ? slots : kMaxCtas));
}

template <int DP, bool BF16>
cudaError_t launch_decode_t(const DecodeArgs& a, int num_sms, int* status, cudaStream_t stream) {
  using C = DecodeCfg<DP>;
  auto kern = decode_kernel<DP, BF16>;
  const int group = a.Hq / a.Hkv, rows = group < kRows ? group : kRows;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  if (e != cudaSuccess) return e;
  const int ctas = decode_ctas(a, C::kCtasPerSm, num_sms);
  e = launch_dependent(kern, ctas, 32 * kWarps, C::kSmemBytes, stream, a, rows, status);
  if (e != cudaSuccess) return e;
  return launch_dependent(decode_join_kernel<BF16>, static_cast<unsigned>(ctas) * rows, kJoinThreads, 0, stream, a, rows, ctas);
}

}  // namespace

size_t decode_workspace_floats(int batch, int Hq, int Hkv, int D, int table_width, int page_size) {
  const int group = Hq / Hkv, blocks = (group + kRows - 1) / kRows, rows = group < kRows ? group : kRows;
  const long long units = (static_cast<long long>(table_width) * page_size + kUnit - 1) / kUnit;
  const long long most = units * batch * Hkv * blocks;
  const long long ctas = most < kMaxCtas ? most : kMaxCtas;
  return static_cast<size_t>(ctas) * (4 + 2 * rows * (D + 2));
}

cudaError_t launch_decode(const DecodeArgs& a, int dtype, int num_sms, int* status, cudaStream_t stream) {
  if (a.D <= 64)
    return dtype ? launch_decode_t<64, true>(a, num_sms, status, stream) : launch_decode_t<64, false>(a, num_sms, status, stream);
  if (a.D <= 128)
    return dtype ? launch_decode_t<128, true>(a, num_sms, status, stream) : launch_decode_t<128, false>(a, num_sms, status, stream);
  return dtype ? launch_decode_t<256, true>(a, num_sms, status, stream) : launch_decode_t<256, false>(a, num_sms, status, stream);
}

}  // namespace fa2
