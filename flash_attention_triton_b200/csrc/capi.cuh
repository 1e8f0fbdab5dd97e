// What the files with C entry points share.
#pragma once
#include <cstdint>

#include "common.cuh"

namespace fa2 {

// Status word, work counter and SM count of the current device, which must be of compute capability 10.x; binds its
// primary context to the calling thread.  Returns a code of fa2_b200.h or a cudaError_t.
int launch_context(LaunchCtx* ctx);

// Tensor map over a [B, H, N, D] 16-bit tensor with box (box_columns, box_rows, 1, 1).
int encode_map(CUtensorMap* m, const void* base, int dtype, int B, int H, int N, int D, const Strides& st,
               int box_columns, int box_rows, CUtensorMapSwizzle swizzle,
               CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
// The same with box (chunk, box_rows, 1, 1).  The chunk
// follows the padded head dim, so for D = 48 or 96 the last box of a row hangs over the
// tensor: those columns read as zeros and are not written.
int make_map(CUtensorMap* m, const void* base, int dtype, int B, int H, int N, int D, const Strides& st, int box_rows);

// Argument checks of the entry points that take grouped heads: head dim, type, and Hkv dividing Hq.
int check_heads(int Hq, int Hkv, int D, int dtype);
// Strides of a dimension of `size` entries above `last` contiguous elements.
inline bool stride_ok(long long stride, int size, int last) {
  return size <= 1 || (stride >= last && stride % 8 == 0 && stride < (1ll << 38));
}

inline bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace fa2
