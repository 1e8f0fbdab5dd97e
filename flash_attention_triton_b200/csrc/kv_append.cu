// New keys and values into the pages of a cache, the position rotation of keys and queries applied on the way.
//
// Token i of sequence s stands at position p = lengths[s] - (tokens of s in this call) + i; its key and value go to
// slot p % page_size of page block_table[s][p / page_size].  The rotation turns the pair (x1, x2) of columns
// (j, j + R/2), or (2j, 2j + 1) interleaved, by the angle whose cosine and sine the tables hold at [p][j]:
//     (x1 cos - x2 sin, x2 cos + x1 sin),  in fp32, rounded once.
//
// Bound by memory for prompts (every element is read once and written once) and by latency for single tokens.
// A thread has one place of the heads' columns for good and takes four 16-byte pieces of one token at a time: the two pieces
// that the rotation joins in two heads, or the same piece in four.  Their loads are in flight together, and the cosines and
// sines are read once for all of them.  Many small CTAs: one loads while others look up places or store.  The first
// warp of a CTA finds sequence, position and page of the CTA's tokens and leaves them in shared memory.
// 31 323 tokens of 32 + 8 + 8 heads of 128 columns: 137 us, 92 % of the measured copy rate (on new inputs every call 145, 87 %); with one head a thread, each token
// behind the stores of the one before, 183 us, with 512 threads to a CTA 178 us, five and six CTAs of 256 threads on an SM
// (48 and 40 registers, spilled) 148 and 161 us; with the first token's loads in front of the look-up, which then waits behind
// those of the whole SM, 184 us.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace fa2 {
namespace {

constexpr int kMaxTokens = 32;  // of one CTA: one lane of the first warp for each

struct TokenPlace {
  long long k, v;  // element offset of the slot in the caches, -1: this token is not written
  int position;    // row of the rotation tables; negative: none
};

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& a, float (&x)[8]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if constexpr (BF16)
      f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    else
      f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
}

__device__ __forceinline__ uint4 load16(const void* base, long long element) {
  return ld_global(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + element));
}
__device__ __forceinline__ void store16(void* base, long long element, const uint4& v) {
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + element) = v;
}

// The sequence of a row: the first s with cu_seqlens[s + 1] > row, `batch` behind the last.  A warp looks at 32 places at once.
__device__ __forceinline__ int sequence_of(const int* cu_seqlens, int batch, int row, int lane) {
  int low = 0, high = batch;
  while (low < high) {
    const int step = (high - low + 31) / 32;
    const int at = min(low + (lane + 1) * step, high);  // cu_seqlens[at] <= row: the answer is at least `at`
    const int below = __popc(__ballot_sync(0xffffffffu, low + lane * step < high && ld_global(cu_seqlens + at) <= row));
    high = min(low + (below + 1) * step, high) - 1;
    low = min(low + below * step, high + 1);
    if (step == 1) break;
  }
  return low;
}

// A sequence of a call has rows that the call has.
__device__ __forceinline__ bool bounds_ok(int start, int end, int tokens) { return start >= 0 && start <= end && end <= tokens; }

// How threads share a token's row: first those with a pair of pieces in the heads of q and k (q's heads first), then those
// with a single piece there, then those with a piece in the heads of v.  Of the threads that have the same place, j of
// `groups` takes heads j, j + groups, ..
constexpr int kPieces = 4;
struct AppendShares {
  int pairs, singles;  // places of a head of q or k
  int pair_groups, single_groups, v_groups;
  int threads;
  explicit AppendShares(const AppendArgs& a) {
    const int heads = (a.q ? a.Hq : 0) + a.Hkv;
    pairs = a.interleaved ? 0 : a.rotary / 16;
    singles = a.D / 8 - 2 * pairs;
    pair_groups = (heads + kPieces / 2 - 1) / (kPieces / 2);
    single_groups = (heads + kPieces - 1) / kPieces;
    v_groups = (a.Hkv + kPieces - 1) / kPieces;
    threads = pairs * pair_groups + singles * single_groups + a.D / 8 * v_groups;
  }
};

constexpr int kMostThreads = 128, kCtasPerSm = 8;

template <bool BF16>
__global__ void __launch_bounds__(kMostThreads, kCtasPerSm)
    kv_append_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ AppendShares shares, int tokens_per_cta, int slices,
                     int* status) {
  __shared__ TokenPlace places[kMaxTokens];
  const int first = blockIdx.x / slices * tokens_per_cta, slice = blockIdx.x % slices;
  const int count = min(tokens_per_cta, a.tokens - first);
  grid_wait_previous();  // and no grid_allow_next, for the reason at decode_join_kernel
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, row = first + lane;
    int sequence = row, fresh = 1, index = 0, length = 0;
    bool inside = lane < count;
    if (a.cu_seqlens == nullptr) {
      if (inside) length = ld_global(a.lengths + sequence);
    } else if (a.batch <= 32) {
      // a sequence a lane, all that there is to know about it asked for at once; each lane then finds its row's (31 323 tokens in 16
      // prompts 141.5 -> 138.9 us, 10 855 in 12 27.3 -> 26.2 against the search below)
      const bool there = lane < a.batch;
      const int start = there ? ld_global(a.cu_seqlens + lane) : 0, end = there ? ld_global(a.cu_seqlens + lane + 1) : 0;
      if (blockIdx.x == 0 && !bounds_ok(start, end, a.tokens)) atomicCAS(status, 0, kStatusSequences | kSiteAppend);
      const int size = there ? ld_global(a.lengths + lane) : 0;
      // the first whose end is behind the CTA's first row, and on from there
      const unsigned behind = __ballot_sync(0xffffffffu, there && end > first);
      sequence = behind ? __ffs(behind) - 1 : a.batch;
      for (int s = sequence; s < a.batch; ++s) {
        const int end_of = __shfl_sync(0xffffffffu, end, s);
        if (inside && sequence == s && end_of <= row) ++sequence;
        if (!__any_sync(0xffffffffu, inside && sequence > s)) break;
      }
      inside = inside && sequence < a.batch;
      const int from = min(sequence, a.batch - 1);
      const int start_of = __shfl_sync(0xffffffffu, start, from);
      fresh = __shfl_sync(0xffffffffu, end, from) - start_of;
      length = __shfl_sync(0xffffffffu, size, from);
      index = row - start_of;
      inside = inside && index >= 0 && bounds_ok(start_of, start_of + fresh, a.tokens);
    } else {
      sequence = sequence_of(a.cu_seqlens, a.batch, first, lane);
      if (inside && sequence < a.batch && ld_global(a.cu_seqlens + sequence + 1) <= row) {  // a later sequence begins in between
        int low = sequence + 1, high = a.batch;
        while (low < high) {
          const int mid = (low + high) >> 1;
          if (ld_global(a.cu_seqlens + mid + 1) <= row) low = mid + 1; else high = mid;
        }
        sequence = low;
      }
      inside = inside && sequence < a.batch;
      if (inside) {
        const int start = ld_global(a.cu_seqlens + sequence);
        length = ld_global(a.lengths + sequence);
        fresh = ld_global(a.cu_seqlens + sequence + 1) - start;
        index = row - start;
        inside = index >= 0 && bounds_ok(start, start + fresh, a.tokens);
      }
      for (int i = blockIdx.x * 32 + lane; i < a.batch; i += gridDim.x * 32)  // what none of these tokens sees, a share for each CTA
        if (!bounds_ok(ld_global(a.cu_seqlens + i), ld_global(a.cu_seqlens + i + 1), a.tokens)) atomicCAS(status, 0, kStatusSequences | kSiteAppend);
    }
    TokenPlace place{-1, -1, -1};
    if (inside) {
      const long long position = static_cast<long long>(length) - fresh + index;
      if (position >= 0) {
        const bool fits = position <= 0x7fffffff;  // (not where cu_seqlens fall)
        const int p = fits ? static_cast<int>(position) : 0, page_index = p / a.page_size;
        int page = -1;
        if (fits && page_index < a.table_width && (a.rotary == 0 || p < a.positions))
          page = ld_global(a.block_table + sequence * a.table_stride + page_index);
        if (page >= 0 && page < a.pages) {
          const long long slot = p - page_index * a.page_size;
          place.k = page * a.sk_cache.page + slot * a.sk_cache.slot;
          place.v = page * a.sv_cache.page + slot * a.sv_cache.slot;
          place.position = p;
        } else {
          atomicCAS(status, 0, kStatusPage | kSiteAppend);
        }
      }
    }
    places[lane] = place;
  }
  __syncthreads();

  // This thread's token among those that the CTA has at a time, and its place in the row.
  const int at = slice * blockDim.x + threadIdx.x;
  const int beside = slices > 1 ? 1 : blockDim.x / shares.threads;
  const int mine = at / shares.threads;
  if (mine >= beside) return;
  int unit = at - mine * shares.threads;
  const int pair_threads = shares.pairs * shares.pair_groups, single_threads = shares.singles * shares.single_groups;
  const bool pair = unit < pair_threads, is_v = unit >= pair_threads + single_threads;
  unit -= pair ? 0 : (is_v ? pair_threads + single_threads : pair_threads);
  const int units = pair ? shares.pairs : (is_v ? a.D / 8 : shares.singles);
  const int groups = pair ? shares.pair_groups : (is_v ? shares.v_groups : shares.single_groups);
  const int group = unit / units;
  unit -= group * units;
  const int hq = a.q != nullptr ? a.Hq : 0, heads = is_v ? a.Hkv : hq + a.Hkv;
  const bool turns = pair || (!is_v && a.interleaved && unit < a.rotary / 8);
  const int column = (pair || is_v ? unit : 2 * shares.pairs + unit) * 8;
  const int half = a.rotary / 2, angle = pair ? unit * 8 : unit * 4;

  for (int t = mine; t < count; t += beside) {
    const long long row = first + t;
    const TokenPlace place = places[t];
    // piece i: which head (below 0: none), and its column
    auto head_of = [&](int i) {
      const int head = group + (pair ? i >> 1 : i) * groups;
      return head < heads ? head : -1;
    };
    auto column_of = [&](int i) { return pair && (i & 1) ? column + half : column; };
    uint4 x[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int head = head_of(i);
      if (head < 0) continue;
      const bool is_q = !is_v && head < hq;
      const void* const src = is_v ? a.v : (is_q ? a.q : a.k);
      const long long row_stride = is_v ? a.sv.row : (is_q ? a.sq.row : a.sk.row), head_stride = is_v ? a.sv.head : (is_q ? a.sq.head : a.sk.head);
      x[i] = load16(src, row * row_stride + (is_q || is_v ? head : head - hq) * head_stride + column_of(i));
    }
    if (turns && place.position >= 0) {
      const float4* const cos = reinterpret_cast<const float4*>(a.cos + static_cast<long long>(place.position) * half + angle);
      const float4* const sin = reinterpret_cast<const float4*>(a.sin + static_cast<long long>(place.position) * half + angle);
      const float4 c0 = ld_global(cos), s0 = ld_global(sin);
      if (pair) {
        const float4 c1 = ld_global(cos + 1), s1 = ld_global(sin + 1);
        const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < kPieces; i += 2) {
          float f[8], g[8];
          unpack8<BF16>(x[i], f);
          unpack8<BF16>(x[i + 1], g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x1 = f[e], x2 = g[e];
            f[e] = x1 * c[e] - x2 * s[e];
            g[e] = x2 * c[e] + x1 * s[e];
          }
          x[i] = pack8<BF16>(f);
          x[i + 1] = pack8<BF16>(g);
        }
      } else {
        const float c[4] = {c0.x, c0.y, c0.z, c0.w}, s[4] = {s0.x, s0.y, s0.z, s0.w};
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          float f[8];
          unpack8<BF16>(x[i], f);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x1 = f[2 * e], x2 = f[2 * e + 1];
            f[2 * e] = x1 * c[e] - x2 * s[e];
            f[2 * e + 1] = x2 * c[e] + x1 * s[e];
          }
          x[i] = pack8<BF16>(f);
        }
      }
    }
    const long long slot = is_v ? place.v : place.k;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int head = head_of(i);
      if (head < 0) continue;
      const bool is_q = !is_v && head < hq;
      const int h = is_q || is_v ? head : head - hq;
      if (!is_q && slot >= 0)
        store16(is_v ? a.v_cache : a.k_cache, slot + h * (is_v ? a.sv_cache.head : a.sk_cache.head) + column_of(i), x[i]);
      void* const dense = is_q ? a.q_out : (is_v ? nullptr : a.k_out);
      if (dense != nullptr)
        store16(dense, (row * (is_q ? a.Hq : a.Hkv) + h) * a.D + column_of(i), slot < 0 ? make_uint4(0, 0, 0, 0) : x[i]);
    }
  }
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, int dtype, int num_sms, int* status, cudaStream_t stream) {
  const AppendShares shares(a);
  const int slices = (shares.threads + kMostThreads - 1) / kMostThreads;  // CTAs beside each other on a token
  // Tokens that a CTA has at a time: as many as there are threads for, few where there are few, so that every SM has some;
  // and in all, so that there are several times as many CTAs as run at once.
  const int fit = slices > 1 ? 1 : kMostThreads / shares.threads, spread = (a.tokens + num_sms - 1) / num_sms;
  const int beside = std::min({fit, spread, kMaxTokens});
  const int threads = ((slices > 1 ? (shares.threads + slices - 1) / slices : beside * shares.threads) + 31) / 32 * 32;
  const int wanted = static_cast<int>((static_cast<long long>(a.tokens) * slices + 48 * num_sms - 1) / (48 * num_sms));
  const int per_cta = std::min((wanted + beside - 1) / beside * beside, kMaxTokens / beside * beside);
  const unsigned grid = static_cast<unsigned>((a.tokens + per_cta - 1) / per_cta) * slices;
  return dtype ? launch_dependent(kv_append_kernel<true>, grid, threads, 0, stream, a, shares, per_cta, slices, status)
               : launch_dependent(kv_append_kernel<false>, grid, threads, 0, stream, a, shares, per_cta, slices, status);
}

}  // namespace fa2
