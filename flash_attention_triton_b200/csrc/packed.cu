// What the attention kernels of packed sequences need beside themselves: the plan of their tiles, the row statistics of
// the backward, and zeros in the rows that belong to no sequence.
#include "packed.cuh"

namespace fa2 {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBins = 1024;

// Whether cu_seqlens rises from 0 or more to at most `rows` (whole CTA).
__device__ bool sequences_ok(const int* cu_seqlens, int batch, int rows) {
  int bad = 0;
  for (int i = threadIdx.x; i <= batch; i += blockDim.x) {
    const int c = ld_global(cu_seqlens + i);
    bad |= c < 0 || c > rows || (i > 0 && c < ld_global(cu_seqlens + i - 1));
  }
  return !__syncthreads_or(bad);
}

// Inclusive sums over the CTA's threads; `total` gets the last one.
__device__ int block_scan(int x, int* shared, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = x;
  __syncthreads();
  int s = shared[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, warp == 0 ? 0 : warp - 1);
  return x + (warp == 0 ? 0 : before);
}

// A list of entries of `per` tiles each, those that start at the highest tiles first: a counting sort by the number
// of the entry in its sequence, in up to 1024 bins.  Entries of one bin stand in any order, which changes no result.
__device__ int write_list(const int* cu_seqlens, int batch, int per, PackedTile* list, int longest, int* full, int* rest,
                          int* cursor, int* shared) {
  const int entries = (longest + per - 1) / per;
  int shift = 0;
  while ((entries - 1) >> shift >= kBins) ++shift;
  full[threadIdx.x] = rest[threadIdx.x] = 0;  // sequences whose bins end before this one; entries of the last bins
  __syncthreads();
  for (int b = threadIdx.x; b < batch; b += kPlanThreads) {
    const int tiles = (ld_global(cu_seqlens + b + 1) - ld_global(cu_seqlens + b) + 127) >> 7, n = (tiles + per - 1) / per;
    if (n >> shift) atomicAdd(full + (n >> shift) - 1, 1);
    if (n & ((1 << shift) - 1)) atomicAdd(rest + (n >> shift), n & ((1 << shift) - 1));
  }
  __syncthreads();
  // thread i has bin 1023 - i: sums from the heaviest bin on
  const int bin = kBins - 1 - threadIdx.x;
  int all, sequences = block_scan(full[bin], shared, all);
  const int mine = (sequences << shift) + rest[bin];
  const int upto = block_scan(mine, shared, all);
  cursor[bin] = upto - mine;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  int before = 0;  // tiles of the sequences so far
  for (int b0 = 0; b0 < batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    const int start = b < batch ? ld_global(cu_seqlens + b) : 0, length = b < batch ? ld_global(cu_seqlens + b + 1) - start : 0;
    const int tiles = (length + 127) >> 7;
    int sum;
    const int base = before + block_scan(tiles, shared, sum) - tiles;
    before += sum;
    // a warp writes the sequences of its 32 lanes, one after the other
    for (int l = 0; l < 32; ++l) {
      const PackedTile e{__shfl_sync(0xffffffffu, start, l), __shfl_sync(0xffffffffu, length, l), 0, __shfl_sync(0xffffffffu, base, l)};
      const int n = (((e.length + 127) >> 7) + per - 1) / per;
      for (int k = lane; k << shift < n; k += 32) {
        const int count = min(n - (k << shift), 1 << shift);
        const int at = atomicAdd(cursor + k, count);
        for (int i = 0; i < count; ++i) {
          *reinterpret_cast<int4*>(list + at + i) = make_int4(e.row0, e.length, ((k << shift) + count - 1 - i) * per, e.base);
        }
      }
    }
  }
  __syncthreads();
  return all;
}

// CTA 0 writes the plan, the others clear the rows of `out` that no sequence has.
__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const int* cu_seqlens, PackedPlan plan, int batch, int rows,
                                                                  bool pairs, void* out, long long row16, int* status) {
  __shared__ int full[kBins], rest[kBins], cursor[kBins], shared[32], longest;
  grid_wait_previous();
  grid_allow_next();
  if (blockIdx.x == 0 && batch <= 32) {
    write_short_plan(ShortBatch(cu_seqlens, batch, rows), plan, pairs, threadIdx.x >> 5, kPlanThreads / 32, status);
    return;
  }
  constexpr int kSome = 8;  // sequences of a lane
  if (blockIdx.x == 0 && batch <= 32 * kSome) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int start[kSome], length[kSome], base[kSome], before = 0;
    bool ok = true;
#pragma unroll
    for (int k = 0; k < kSome; ++k) {
      const int b = k * 32 + lane;
      start[k] = b < batch ? ld_global(cu_seqlens + b) : 0;
      length[k] = b < batch ? ld_global(cu_seqlens + b + 1) : 0;  // its end, as yet
    }
#pragma unroll
    for (int k = 0; k < kSome; ++k) ok &= start[k] >= 0 && length[k] >= start[k] && length[k] <= rows;
    ok = __all_sync(0xffffffffu, ok);
#pragma unroll
    for (int k = 0; k < kSome; ++k) {
      length[k] = ok ? length[k] - start[k] : 0;
      const int tiles = (length[k] + 127) >> 7;
      int upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      base[k] = before + upto - tiles;
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    const int tiles = write_list_by_ballots<kSome>(start, length, base, 1, plan.tiles, warp, kPlanThreads / 32);
    const int two = pairs ? write_list_by_ballots<kSome>(start, length, base, 2, plan.pairs, warp, kPlanThreads / 32) : 0;
    if (threadIdx.x == 0) {
      plan.counts[0] = tiles;
      plan.counts[1] = two;
      plan.counts[2] = 0;
      if (!ok) atomicCAS(status, 0, kStatusSequences);
    }
    return;
  }
  const bool ok = sequences_ok(cu_seqlens, batch, rows);
  if (blockIdx.x > 0) {
    const int first = ok ? ld_global(cu_seqlens) : rows, last = ok ? ld_global(cu_seqlens + batch) : rows;
    clear_outside(out, row16, first, last, rows, (blockIdx.x - 1ll) * kPlanThreads + threadIdx.x, (gridDim.x - 1ll) * kPlanThreads);
    return;
  }
  if (threadIdx.x == 0) longest = 0;
  __syncthreads();
  int most = 0;
  if (ok)
    for (int b = threadIdx.x; b < batch; b += kPlanThreads)
      most = max(most, (ld_global(cu_seqlens + b + 1) - ld_global(cu_seqlens + b) + 127) >> 7);
  most = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(most));
  if ((threadIdx.x & 31) == 0 && most > 0) atomicMax(&longest, most);
  __syncthreads();
  int counts[2] = {0, 0};
  if (longest > 0) {
    counts[0] = write_list(cu_seqlens, batch, 1, plan.tiles, longest, full, rest, cursor, shared);
    if (pairs) counts[1] = write_list(cu_seqlens, batch, 2, plan.pairs, longest, full, rest, cursor, shared);
  }
  if (threadIdx.x == 0) {
    plan.counts[0] = counts[0];
    plan.counts[1] = counts[1];
    plan.counts[2] = 0;
    if (!ok) atomicCAS(status, 0, kStatusSequences);
  }
}

// ----------------------------------------------------------------------------------------
// Backward preprocess: delta = rowsum(dO o O), with -lse log2(e) (+ kProbabilityPower) by tile.  Bound by reading O and dO once.  A CTA takes
// eight heads of 32 rows of a tile, which lie one behind the other in memory; D / 8 adjacent lanes add up
// one head of one row in a fixed order.  23 202 rows, 16 heads of 128 columns: 41.8 us for 192 MB read, 70 % of the measured copy rate.
// ----------------------------------------------------------------------------------------
constexpr int kPreThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPreHeads = 8;  // of a CTA

template <bool BF16>
__device__ __forceinline__ float2 both(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPreThreads) packed_preprocess_kernel(
    const PackedTile* tiles, const int* counts, int capacity, const int* cu_seqlens, const uint16_t* o, const uint16_t* dout,
    RowStrides sdo, const float* lse, PackedStats out, int rows, int batch, int Hq, int Hkv, int Dg, void* dq, void* dk, void* dv) {
  constexpr int kLanes = D / 8, kGroups = kPreThreads / kLanes;
  __shared__ float delta[kPreHeads][33];
  __shared__ unsigned amax[kPreHeads];
  grid_wait_previous();
  grid_allow_next();
  if (blockIdx.x == 0 && threadIdx.x == 0) *out.written = 0;
  const int parts = 4 * ((Hq + kPreHeads - 1) / kPreHeads);  // CTAs of a tile
  const int entry = blockIdx.x / parts, part = blockIdx.x - entry * parts;
  // (asked for together: an entry behind the last one may hold anything)
  const int count = ld_global(counts), start = ld_global(cu_seqlens), end = ld_global(cu_seqlens + batch);
  const PackedTile e = load_tile(tiles + entry);
  // rows of the gradients that no sequence has
  {
    const int first = count ? start : rows, last = count ? end : rows;
    const long long worker = static_cast<long long>(blockIdx.x) * kPreThreads + threadIdx.x, workers = static_cast<long long>(gridDim.x) * kPreThreads;
    clear_outside(dq, static_cast<long long>(Hq) * Dg / 8, first, last, rows, worker, workers);
    clear_outside(dk, static_cast<long long>(Hkv) * Dg / 8, first, last, rows, worker, workers);
    clear_outside(dv, static_cast<long long>(Hkv) * Dg / 8, first, last, rows, worker, workers);
  }
  if (entry >= count) return;
  const int quarter = part & 3, h0 = part / 4 * kPreHeads, heads = min(Hq - h0, kPreHeads);
  const int local = e.tile * 128 + quarter * 32;  // first of the 32 rows in the sequence
  const int here = min(max(e.length - local, 0), 32);
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  if (threadIdx.x < kPreHeads) amax[threadIdx.x] = 0;
  // the result that this thread writes at the end
  static_assert(kPreHeads * 32 == kPreThreads, "one result a thread");
  const int out_h = threadIdx.x / 32, out_r = threadIdx.x % 32;
  const bool writes = out_h < heads, inside = writes && out_r < here;
  const float row_lse = inside ? ld_global(lse + static_cast<size_t>(h0 + out_h) * rows + e.row0 + local + out_r) : 0.f;
  __syncthreads();
  const int work = here * heads;
  for (int i0 = group; i0 < (work + 4 * kGroups - 1) / (4 * kGroups) * (4 * kGroups); i0 += 4 * kGroups) {
    uint4 a[4], b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kGroups, r = i / heads, h = h0 + i - r * heads;
      a[u] = b[u] = make_uint4(0, 0, 0, 0);
      if (i < work && lane * 8 < Dg) {
        const long long row = e.row0 + local + r;
        a[u] = ld_global(reinterpret_cast<const uint4*>(o + (row * Hq + h) * Dg + lane * 8));
        b[u] = ld_global(reinterpret_cast<const uint4*>(dout + row * sdo.row + h * sdo.head + lane * 8));
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kGroups, r = i / heads, h = i - r * heads;
      const uint32_t x[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, y[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
      float sum = 0.f;
      unsigned most = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 f = both<BF16>(x[w]), g = both<BF16>(y[w]);
        sum = fmaf(f.x, g.x, sum);
        sum = fmaf(f.y, g.y, sum);
        if constexpr (!BF16) most = max(most, max(y[w] & 0x7fffu, (y[w] >> 16) & 0x7fffu));
      }
#pragma unroll
      for (int s = kLanes / 2; s > 0; s >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if constexpr (!BF16) most = max(most, __shfl_xor_sync(0xffffffffu, most, s));
      }
      if (lane == 0 && i < work) {
        delta[h][r] = sum;
        if constexpr (!BF16) atomicMax(amax + h, most);
      }
    }
  }
  __syncthreads();
  if (!writes) return;
  const int h = h0 + out_h;
  float* const to = out.stats + (static_cast<size_t>(h) * capacity + e.base + e.tile) * 256 + quarter * 32 + out_r;
  to[0] = inside ? kProbabilityPower<BF16> - row_lse * kLog2e : -INFINITY;
  to[128] = inside ? -delta[out_h][out_r] : 0.f;
  if (!BF16 && out_r == 0)
    out.amax[(static_cast<size_t>(h) * capacity + e.base + e.tile) * 4 + quarter] = amax[out_h];
}

}  // namespace

cudaError_t launch_packed_plan(const PackedShape& s, const int* cu_seqlens, const PackedPlan& plan, bool pairs, void* out,
                               int* status, int num_sms, cudaStream_t stream) {
  // a few CTAs beside the plan: a buffer of fixed size may have many rows behind its last sequence
  const long long row16 = static_cast<long long>(s.Hq) * s.Dg / 8;
  const long long wanted = (s.rows * row16 + 64 * kPlanThreads - 1) / (64 * kPlanThreads);
  const unsigned grid = 1 + static_cast<unsigned>(wanted < num_sms ? wanted : num_sms);
  return launch_dependent(packed_plan_kernel, grid, kPlanThreads, 0, stream, cu_seqlens, plan, s.batch, s.rows, pairs, out, row16, status);
}

template <int D>
static cudaError_t launch_preprocess_t(const PackedShape& s, const PackedPlan& plan, const int* cu_seqlens, const void* o,
                                       const void* dout, const RowStrides& sdo, const float* lse, const PackedStats& stats,
                                       void* dq, void* dk, void* dv, cudaStream_t stream) {
  auto kern = s.dtype ? packed_preprocess_kernel<D, true> : packed_preprocess_kernel<D, false>;
  return launch_dependent(kern, 4u * plan.capacity * ((s.Hq + kPreHeads - 1) / kPreHeads), kPreThreads, 0, stream, plan.tiles, plan.counts, plan.capacity, cu_seqlens,
                          static_cast<const uint16_t*>(o), static_cast<const uint16_t*>(dout), sdo, lse, stats, s.rows, s.batch, s.Hq,
                          s.Hkv, s.Dg, dq, dk, dv);
}

cudaError_t launch_packed_preprocess(const PackedShape& s, const PackedPlan& plan, const int* cu_seqlens, const void* o,
                                     const void* dout, const RowStrides& sdo, const float* lse, const PackedStats& stats,
                                     void* dq, void* dk, void* dv, cudaStream_t stream) {
  if (s.D == 32) return launch_preprocess_t<32>(s, plan, cu_seqlens, o, dout, sdo, lse, stats, dq, dk, dv, stream);
  if (s.D == 64) return launch_preprocess_t<64>(s, plan, cu_seqlens, o, dout, sdo, lse, stats, dq, dk, dv, stream);
  return launch_preprocess_t<128>(s, plan, cu_seqlens, o, dout, sdo, lse, stats, dq, dk, dv, stream);
}

}  // namespace fa2
