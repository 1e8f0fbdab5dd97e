// New keys and values into the pages of a cache, the position rotation of keys and queries applied on the way.
//
// Token i of sequence s stands at position p = lengths[s] - (tokens of s in this call) + i; its key and value go to
// slot p % page_size of page block_table[s][p / page_size].  The rotation turns the pair (x1, x2) of columns
// (j, j + R/2), or (2j, 2j + 1) interleaved, by the angle whose cosine and sine the tables hold at [p][j]:
//     (x1 cos - x2 sin, x2 cos + x1 sin),  in fp32, rounded once.
//
// Bound by memory for prompts (every element is read once and written once) and by latency for single tokens.
// A thread has one place of a token's row for good: 16 bytes of one head, or the two 16-byte pieces that the
// rotation joins; the token loop around it only adds strides.  A warp of the CTA finds sequence, position and
// page of the CTA's tokens once (one binary search per token) and leaves them in shared memory.
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

template <bool BF16>
__global__ void __launch_bounds__(512) kv_append_kernel(const __grid_constant__ AppendArgs a, int tokens_per_cta,
                                                        int* status) {
  __shared__ TokenPlace places[kMaxTokens];
  const int first = blockIdx.x * tokens_per_cta;
  const int count = min(tokens_per_cta, a.tokens - first);
  grid_wait_previous();
  grid_allow_next();
  if (threadIdx.x < count) {
    const int row = first + threadIdx.x;
    int sequence = row, fresh = 1, index = 0;
    bool inside = true;
    if (a.cu_seqlens != nullptr) {
      // the last sequence that starts at or before this row
      int low = 0, high = a.batch;
      while (low < high) {
        const int mid = (low + high) >> 1;
        if (ld_global(a.cu_seqlens + mid + 1) <= row) low = mid + 1; else high = mid;
      }
      sequence = low;
      inside = sequence < a.batch;
      if (inside) {
        const int start = ld_global(a.cu_seqlens + sequence);
        fresh = ld_global(a.cu_seqlens + sequence + 1) - start;
        index = row - start;
        inside = index >= 0;
      }
    }
    TokenPlace place{-1, -1, -1};
    if (inside) {
      const long long position = static_cast<long long>(ld_global(a.lengths + sequence)) - fresh + index;
      if (position >= 0) {
        const long long page_index = position / a.page_size;
        int page = -1;
        if (page_index < a.table_width && (a.rotary == 0 || position < a.positions))
          page = ld_global(a.block_table + sequence * a.table_stride + page_index);
        if (page >= 0 && page < a.pages) {
          const long long slot = position - page_index * a.page_size;
          place.k = page * a.sk_cache.page + slot * a.sk_cache.slot;
          place.v = page * a.sv_cache.page + slot * a.sv_cache.slot;
          place.position = static_cast<int>(position);
        } else {
          atomicCAS(status, 0, kStatusPage | kSiteAppend);
        }
      }
    }
    places[threadIdx.x] = place;
  }
  __syncthreads();

  // This thread's place in a token's row: which tensor, head, and which piece or pair of pieces.
  const int d8 = a.D / 8, half8 = a.interleaved ? 0 : a.rotary / 16;  // pieces of half the rotated columns
  const int turned = a.interleaved ? a.rotary / 8 : half8;            // units of a head that the rotation turns
  const int units = d8 - half8;                                       // of a head of q or k; a head of v has d8
  int unit = blockIdx.y * blockDim.x + threadIdx.x;
  const int nq = a.q != nullptr ? a.Hq * units : 0, nk = a.Hkv * units, nv = a.Hkv * d8;
  if (unit >= nq + nk + nv) return;
  const bool is_q = unit < nq, is_v = unit >= nq + nk;
  unit -= is_q ? 0 : (is_v ? nq + nk : nq);
  const int per_head = is_v ? d8 : units;
  const int head = unit / per_head;
  unit -= head * per_head;
  const bool turns = !is_v && unit < turned, pair = turns && !a.interleaved;
  const int column = (!is_v && !a.interleaved && unit >= half8 ? unit + half8 : unit) * 8;
  const void* src = is_q ? a.q : (is_v ? a.v : a.k);
  const RowStrides ss = is_q ? a.sq : (is_v ? a.sv : a.sk);
  const long long from = head * ss.head + column;
  const int other = half8 * 8;  // columns between the two pieces of a pair
  void* const dense = is_q ? a.q_out : (is_v ? nullptr : a.k_out);
  const long long dense_row = static_cast<long long>(is_q ? a.Hq : a.Hkv) * a.D;
  const long long dense_at = static_cast<long long>(head) * a.D + column;
  void* const cache = is_q ? nullptr : (is_v ? a.v_cache : a.k_cache);
  const long long cache_at = head * (is_v ? a.sv_cache : a.sk_cache).head + column;

#pragma unroll 4
  for (int t = 0; t < count; ++t) {
    const long long row = first + t;
    const TokenPlace place = places[t];
    uint4 x = load16(src, row * ss.row + from), y{};
    if (pair) y = load16(src, row * ss.row + from + other);
    if (turns && place.position >= 0) {
      const int half = a.rotary / 2;
      const float* cos = a.cos + static_cast<long long>(place.position) * half;
      const float* sin = a.sin + static_cast<long long>(place.position) * half;
      float f[8], g[8];
      unpack8<BF16>(x, f);
      if (pair) {
        unpack8<BF16>(y, g);
        const int j = unit * 8;
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 c4 = ld_global(reinterpret_cast<const float4*>(cos + j + i));
          const float4 s4 = ld_global(reinterpret_cast<const float4*>(sin + j + i));
          const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x1 = f[i + e], x2 = g[i + e];
            f[i + e] = x1 * c[e] - x2 * s[e];
            g[i + e] = x2 * c[e] + x1 * s[e];
          }
        }
        y = pack8<BF16>(g);
      } else {
        const int j = unit * 4;
        const float4 c4 = ld_global(reinterpret_cast<const float4*>(cos + j));
        const float4 s4 = ld_global(reinterpret_cast<const float4*>(sin + j));
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x1 = f[2 * e], x2 = f[2 * e + 1];
          f[2 * e] = x1 * c[e] - x2 * s[e];
          f[2 * e + 1] = x2 * c[e] + x1 * s[e];
        }
      }
      x = pack8<BF16>(f);
    }
    const long long slot = is_v ? place.v : place.k;
    if (cache != nullptr && slot >= 0) {
      store16(cache, slot + cache_at, x);
      if (pair) store16(cache, slot + cache_at + other, y);
    }
    if (dense != nullptr) {
      if (slot < 0) x = y = make_uint4(0, 0, 0, 0);
      store16(dense, row * dense_row + dense_at, x);
      if (pair) store16(dense, row * dense_row + dense_at + other, y);
    }
  }
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, int dtype, int num_sms, int* status, cudaStream_t stream) {
  const int d8 = a.D / 8, units = d8 - (a.interleaved ? 0 : a.rotary / 16);
  const int places = (a.q != nullptr ? a.Hq * units : 0) + a.Hkv * (units + d8);
  const int slices = (places + 511) / 512;                                  // CTAs beside each other on a token
  const int threads = ((places + slices - 1) / slices + 31) / 32 * 32;
  const long long wanted = (static_cast<long long>(a.tokens) * slices + 8 * num_sms - 1) / (8ll * num_sms);
  const int per_cta = static_cast<int>(wanted < 1 ? 1 : (wanted > kMaxTokens ? kMaxTokens : wanted));
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((a.tokens + per_cta - 1) / per_cta, slices);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return dtype ? cudaLaunchKernelEx(&cfg, kv_append_kernel<true>, a, per_cta, status)
               : cudaLaunchKernelEx(&cfg, kv_append_kernel<false>, a, per_cta, status);
}

}  // namespace fa2
