// Arguments of the kernels that work on a paged key-value cache: tensors [pages, page_size, Hkv, D] whose pages a
// block table [batch, table_width] hands out to the sequences.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace fa2 {

// Status word of a kernel that met a page outside the cache, or a position beyond the block table or the rotation
// tables: what it stands for is neither read nor written.
constexpr int kStatusPage = 0x40000;
// Status word of cu_seqlens that fall, or leave the rows: every output of the attention is zero then; the append leaves out the tokens of
// sequences that leave the rows.
constexpr int kStatusSequences = 0x80000;
enum PagedSite { kSiteAppend = 1, kSiteDecode };

// Element strides; the last dimension is contiguous.
struct RowStrides {
  long long row, head;
};
struct CacheStrides {
  long long page, slot, head;
};

struct AppendArgs {
  const void *q, *k, *v;  // [tokens, H, D]; q may be null
  void *q_out, *k_out;    // dense [tokens, H, D]; k_out may be null
  void *k_cache, *v_cache;
  const int* block_table;
  const int* lengths;     // [batch]: tokens of a sequence in the cache, those of this call included
  const int* cu_seqlens;  // [batch + 1], or null: token i is the one new token of sequence i
  const float *cos, *sin; // [positions, rotary / 2]
  RowStrides sq, sk, sv;
  CacheStrides sk_cache, sv_cache;
  long long table_stride;
  int tokens, batch, Hq, Hkv, D, pages, page_size, table_width, positions, rotary, interleaved;
};
cudaError_t launch_kv_append(const AppendArgs& a, int dtype, int num_sms, int* status, cudaStream_t stream);

struct DecodeArgs {
  const void* q;  // [batch, Hq, D]
  const void *k_cache, *v_cache;
  void* out;      // dense [batch, Hq, D]
  const int* block_table;
  const int* lengths;  // [batch]: keys of a sequence, 2^31 - 1: all that the block table has room for; out is zero where there are none
  float* workspace;    // partial results, decode_workspace_floats()
  RowStrides sq;
  CacheStrides sk_cache, sv_cache;
  long long table_stride;
  int batch, Hq, Hkv, D, pages, page_size, table_width;
  float scale_log2;
};
size_t decode_workspace_floats(int batch, int Hq, int Hkv, int D, int table_width, int page_size);
// Rows of the boxes that the cache's tensor maps bring in: the largest part of 16 that divides a page.
int decode_box_rows(int page_size);
// tk, tv: maps (D, slots, heads, pages) with boxes (64, decode_box_rows, 1, 1), 128-byte swizzle.
cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeArgs& a, int dtype, int num_sms, int* status,
                          cudaStream_t stream);

}  // namespace fa2
