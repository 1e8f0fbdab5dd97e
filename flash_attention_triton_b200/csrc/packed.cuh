// Attention over packed sequences: sequences of different lengths one behind the other in [rows, heads, D] tensors,
// cu_seqlens[s] .. cu_seqlens[s + 1] - 1 the rows of sequence s, and G = Hq / Hkv query heads to a key head.
//
// The kernels work on 128-row tiles of the sequences.  Which tiles there are only the device knows, so a kernel in
// front of them writes the plan: every tile of every sequence, the ones that meet the most tiles first, for the same reason
// as grouped_order in common.cuh.  Tile t of a sequence of n tiles meets t + 1 KV tiles as a Q tile; KV tile n - 1 - t
// meets as many Q tiles, so one order serves both.
//
// What the tensor maps cannot know either is where a sequence ends inside a tile.  Loads bring the rows of the next
// sequence along (or zeros behind the last row): as rows of the result they are not stored, and where they are
// summed over (V; Q and dO for dK and dV; K and V for dQ) the warp that issues the product first clears them in
// shared memory, because 0 x NaN is none.  Stores of 32 rows go through the tensor map where all of them belong
// to the sequence, row by row where not.
#pragma once
#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace fa2 {

// One tile, or two adjacent ones, of a sequence.
struct PackedTile {
  int row0;    // first row of the sequence
  int length;  // its rows
  int tile;    // (first) tile of this entry
  int base;    // number of the sequence's tile 0 among all tiles, in the order of the sequences
};

struct PackedPlan {
  int* counts;         // [0] tiles, [1] pairs of tiles, [2] the forward's work counter, zero behind the plan kernel
  PackedTile* tiles;   // heaviest first, room for `capacity`
  PackedTile* pairs;   // pairs of adjacent tiles, likewise
  int capacity;
};
// Tiles of `rows` rows in `batch` sequences, at most.
inline int packed_capacity(int rows, int batch) { return rows / 128 + batch; }
inline size_t packed_plan_bytes(int rows, int batch) { return 16 + 2 * sizeof(PackedTile) * packed_capacity(rows, batch); }
inline PackedPlan packed_plan(void* p, int rows, int batch) {
  const int n = packed_capacity(rows, batch);
  PackedTile* const tiles = reinterpret_cast<PackedTile*>(static_cast<char*>(p) + 16);
  return PackedPlan{static_cast<int*>(p), tiles, tiles + n, n};
}

struct PackedShape {
  int rows, batch, Hq, Hkv;
  int D;   // head dim the kernels are instantiated for: 32, 64 or 128
  int Dg;  // of the tensors
  int dtype;
  float scale;
};

// The backward's P, from lse and at most 1, carries this power of two at fp16 for the reason at kWeightPower (common.cuh): a key whose
// weights are small in thousands of rows has its dV from them.  It comes with the exponent, and dV and dS give it back: off by 2^-39 at
// most below 2^-28.  2^16, where fp16 ends, leaves 2^2 for the rounding of lse beside scores of millions.
template <bool BF16>
constexpr float kProbabilityPower = BF16 ? 0.0f : 14.0f;  // logarithm to 2
template <bool BF16>
constexpr float kProbabilityInverse = BF16 ? 1.0f : 1.0f / 16384;

// What the backward's preprocess leaves: -lse log2(e) + kProbabilityPower and -delta by tile, [Hq][capacity][2][128], rows behind a
// sequence -inf and 0; at fp16 also the largest |dout| of every 32 rows, [Hq][capacity][4] (see head_dscale).
struct PackedStats {
  float* stats;
  unsigned* amax;
  unsigned* written;  // zero behind the preprocess; 1 once the dK / dV kernel has seen it complete
};
inline size_t packed_stats_bytes(int rows, int batch, int Hq) {
  return static_cast<size_t>(packed_capacity(rows, batch)) * Hq * (256 + 4) * 4 + 16;
}

cudaError_t launch_packed_plan(const PackedShape& s, const int* cu_seqlens, const PackedPlan& plan, bool pairs, void* out,
                               int* status, int num_sms, cudaStream_t stream);
// Whether the forward has no plan kernel in front of it.  Its CTAs then find their items in cu_seqlens by themselves, and it writes the plan for
// the backward and clears what launch_packed_plan would: 2.5 us less on the host, up to 3 on the GPU.
bool packed_fwd_alone(const PackedShape& s, int num_sms);
cudaError_t launch_packed_fwd(const PackedShape& s, const int* cu_seqlens, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                              const CUtensorMap& tv, const CUtensorMap& to, void* out, float* lse, int* status, int num_sms,
                              cudaStream_t stream);
cudaError_t launch_packed_preprocess(const PackedShape& s, const PackedPlan& plan, const int* cu_seqlens, const void* o,
                                     const void* dout, const RowStrides& sdo, const float* lse, const PackedStats& stats,
                                     void* dq, void* dk, void* dv, cudaStream_t stream);
// Rows of a step of a backward kernel with `heads` CTAs to a tile, and the box height of the tensors it walks; of the dK / dV kernel in
// clusters, which are for launches of few CTAs, 128.
int packed_step_rows(const PackedShape& s, int heads, int num_sms);
// CTAs of the dK / dV kernel that share the query heads of a KV tile: 1, 2 or 4, a divisor of G.
int packed_cluster(const PackedShape& s, int num_sms);
cudaError_t launch_packed_dkdv(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                               const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdk, const CUtensorMap& tdv,
                               void* dk, void* dv, const PackedStats& stats, int step_rows, int cluster, int* status,
                               cudaStream_t stream);
cudaError_t launch_packed_dq(const PackedShape& s, const PackedPlan& plan, const CUtensorMap& tq, const CUtensorMap& tk,
                             const CUtensorMap& tv, const CUtensorMap& tdo, const CUtensorMap& tdq, void* dq,
                             const PackedStats& stats, int step_rows, int* status, cudaStream_t stream);

// launch_dependent (common.cuh) in clusters of `cluster` CTAs.
template <typename... Params, typename... Args>
inline cudaError_t launch_dependent_cluster(void (*kernel)(Params...), unsigned grid, unsigned cluster, int threads, int smem_bytes,
                                            cudaStream_t stream, Args&&... args) {
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

#ifdef __CUDACC__
__device__ __forceinline__ PackedTile load_tile(const PackedTile* p) {
  const uint4 v = ld_global(reinterpret_cast<const uint4*>(p));
  return PackedTile{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w)};
}

// A list of entries of `per` tiles each, those that start at the highest tiles first, for up to 32 SEQUENCES sequences, as many
// to a lane: entry t of a sequence comes behind those of higher numbers in all sequences and those of the same number in the
// sequences before it, which each of the `warps` warps counts without a word to the others.  Returns the entries.
template <int SEQUENCES>
__device__ __forceinline__ int write_list_by_ballots(const int (&start)[SEQUENCES], const int (&length)[SEQUENCES],
                                                     const int (&base)[SEQUENCES], int per, PackedTile* list, int warp, int warps) {
  const int lane = threadIdx.x & 31;
  int n[SEQUENCES], all = 0, mine = 0;
#pragma unroll
  for (int k = 0; k < SEQUENCES; ++k) {
    n[k] = ((length[k] + 127) / 128 + per - 1) / per;
    mine = max(mine, n[k]), all += n[k];
  }
  const int most = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(mine));
  for (int t = warp; t < most; t += warps) {
    int higher = 0;
#pragma unroll
    for (int k = 0; k < SEQUENCES; ++k) higher += max(n[k] - t - 1, 0);
    int at = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(higher));
#pragma unroll
    for (int k = 0; k < SEQUENCES; ++k) {
      const unsigned same = __ballot_sync(0xffffffffu, n[k] > t);
      if (n[k] > t) *reinterpret_cast<int4*>(list + at + __popc(same & ((1u << lane) - 1u))) = make_int4(start[k], length[k], t * per, base[k]);
      at += __popc(same);
    }
  }
  return __reduce_add_sync(0xffffffffu, static_cast<unsigned>(all));
}

// Up to 32 sequences, one a lane (whole warp).
struct ShortBatch {
  int start, length;  // of this lane's sequence; all lengths 0 where cu_seqlens fall or leave the rows
  int base;           // tiles of the sequences before it
  bool ok;
  int first, last;    // rows that the sequences cover
  __device__ __forceinline__ ShortBatch(const int* cu_seqlens, int batch, int rows) {
    const int lane = threadIdx.x & 31;
    start = lane < batch ? ld_global(cu_seqlens + lane) : 0;
    const int end = lane < batch ? ld_global(cu_seqlens + lane + 1) : 0;
    ok = __all_sync(0xffffffffu, start >= 0 && end >= start && end <= rows);
    first = ok ? __shfl_sync(0xffffffffu, start, 0) : rows;
    last = ok ? __shfl_sync(0xffffffffu, end, batch - 1) : rows;
    length = ok ? end - start : 0;
    base = (length + 127) >> 7;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, base, o);
      if (lane >= o) base += y;
    }
    base -= (length + 127) >> 7;
  }
};

__device__ __forceinline__ void write_short_plan(const ShortBatch& s, const PackedPlan& plan, bool pairs, int warp, int warps, int* status) {
  const int start[1] = {s.start}, length[1] = {s.length}, base[1] = {s.base};
  const int tiles = write_list_by_ballots<1>(start, length, base, 1, plan.tiles, warp, warps);
  const int two = pairs ? write_list_by_ballots<1>(start, length, base, 2, plan.pairs, warp, warps) : 0;
  if (warp == 0 && (threadIdx.x & 31) == 0) {
    plan.counts[0] = tiles;
    plan.counts[1] = two;
    plan.counts[2] = 0;
    if (!s.ok) atomicCAS(status, 0, kStatusSequences);
  }
}

// Zeros in the rows of a dense [rows, row16 * 8] tensor that no sequence has.
__device__ __forceinline__ void clear_outside(void* out, long long row16, int first, int last, int rows, long long worker, long long workers) {
  if (out == nullptr) return;
  uint4* const p = static_cast<uint4*>(out);
  for (long long i = worker; i < first * row16; i += workers) p[i] = make_uint4(0, 0, 0, 0);
  for (long long i = last * row16 + worker; i < rows * row16; i += workers) p[i] = make_uint4(0, 0, 0, 0);
}

// Clears rows `first` .. ROWS - 1 of a staged [ROWS, D] tile (whole warp; nothing where first >= ROWS) before a product sums
// over them.  A row stays within its own bytes under the swizzle, so the end of every chunk tile is cleared as it lies.
template <int D, int ROWS>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int first, int lane) {
  using T = Tile<D>;
  if (first >= ROWS) return;
  if (first < 0) first = 0;
  __syncwarp();
  for (int ch = 0; ch < T::kChunks; ++ch)
    for (int at = first * T::kRowBytes + lane * 16; at < ROWS * T::kRowBytes; at += 512)
      *reinterpret_cast<uint4*>(tile + ch * (ROWS * T::kRowBytes) + at) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}
#endif

}  // namespace fa2
