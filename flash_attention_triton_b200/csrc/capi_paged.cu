// C entry points of the paged key-value cache: argument checks and launches.
#include <cmath>

#include "../../include/fa2_b200.h"
#include "capi.cuh"
#include "paged.cuh"

namespace fa2 {

int check_heads(int Hq, int Hkv, int D, int dtype) {
  if (D < 8 || D > 256 || D % 8 != 0) return FA2_ERR_HEAD_DIM;
  if (dtype != FA2_DTYPE_FP16 && dtype != FA2_DTYPE_BF16) return FA2_ERR_DTYPE;
  if (Hkv < 1 || Hq < 1 || Hq > 65535) return FA2_ERR_SHAPE;
  return Hq % Hkv ? FA2_ERR_HEADS : FA2_OK;
}

namespace {

int check_cache(int batch, int pages, int page_size, int table_width) {
  if (batch < 1 || batch > (1 << 20) || pages < 1 || page_size < 1 || table_width < 1) return FA2_ERR_SHAPE;
  return static_cast<long long>(table_width) * page_size > 0x7fffffffll ? FA2_ERR_SHAPE : FA2_OK;
}

RowStrides row_strides(const long long* s, int H, int D) {
  return s ? RowStrides{s[0], s[1]} : RowStrides{static_cast<long long>(H) * D, D};
}
CacheStrides cache_strides(const long long* s, int page_size, int H, int D) {
  return s ? CacheStrides{s[0], s[1], s[2]}
           : CacheStrides{static_cast<long long>(page_size) * H * D, static_cast<long long>(H) * D, D};
}
bool rows_ok(const RowStrides& s, int rows, int H, int D) {
  return stride_ok(s.row, rows, D) && stride_ok(s.head, H, D);
}
bool cache_ok(const CacheStrides& s, int pages, int page_size, int H, int D) {
  return stride_ok(s.page, pages, D) && stride_ok(s.slot, page_size, D) && stride_ok(s.head, H, D);
}

}  // namespace
}  // namespace fa2

using namespace fa2;

extern "C" {

int fa2_kv_append(const void* q, const void* k, const void* v, void* q_out, void* k_out, void* k_cache, void* v_cache,
                  const int* block_table, const int* lengths, const int* cu_seqlens, const float* cos, const float* sin,
                  int tokens, int batch, int Hq, int Hkv, int D, int pages, int page_size, int table_width, int positions,
                  int rotary, int interleaved, int dtype, const long long* strides, fa2_stream_t stream) {
  if (!k || !v || !k_cache || !v_cache || !block_table || !lengths || (q != nullptr) != (q_out != nullptr))
    return FA2_ERR_NULL_POINTER;
  if (int e = check_heads(q ? Hq : Hkv, Hkv, D, dtype)) return e;
  if (int e = check_cache(batch, pages, page_size, table_width)) return e;
  if (tokens < 0 || tokens > (1 << 24) || (!cu_seqlens && tokens != batch)) return FA2_ERR_SHAPE;
  if (rotary < 0 || rotary > D || rotary % 16 || (rotary && (!cos || !sin || positions < 1))) return FA2_ERR_ROTARY;
  for (const void* p : {q, k, v, static_cast<const void*>(q_out), static_cast<const void*>(k_out),
                        static_cast<const void*>(k_cache), static_cast<const void*>(v_cache), static_cast<const void*>(cos),
                        static_cast<const void*>(sin)})
    if (!aligned_to(p, 16)) return FA2_ERR_MISALIGNED;
  AppendArgs a{q, k, v, q_out, k_out, k_cache, v_cache, block_table, lengths, cu_seqlens, rotary ? cos : nullptr,
               rotary ? sin : nullptr, row_strides(strides, Hq, D), row_strides(strides ? strides + 2 : nullptr, Hkv, D),
               row_strides(strides ? strides + 4 : nullptr, Hkv, D),
               cache_strides(strides ? strides + 6 : nullptr, page_size, Hkv, D),
               cache_strides(strides ? strides + 9 : nullptr, page_size, Hkv, D), strides ? strides[12] : table_width,
               tokens, batch, q ? Hq : 0, Hkv, D, pages, page_size, table_width, positions, rotary, interleaved != 0};
  if ((q && !rows_ok(a.sq, tokens, Hq, D)) || !rows_ok(a.sk, tokens, Hkv, D) || !rows_ok(a.sv, tokens, Hkv, D) ||
      !cache_ok(a.sk_cache, pages, page_size, Hkv, D) || !cache_ok(a.sv_cache, pages, page_size, Hkv, D) ||
      (batch > 1 && a.table_stride < 0))
    return FA2_ERR_STRIDE;
  if (tokens == 0) return FA2_OK;
  LaunchCtx ctx;
  if (int e = launch_context(&ctx)) return e;
  return static_cast<int>(launch_kv_append(a, dtype, ctx.num_sms, ctx.status, static_cast<cudaStream_t>(stream)));
}

size_t fa2_decode_workspace_bytes(int batch, int Hq, int Hkv, int D, int page_size, int table_width) {
  if (check_heads(Hq, Hkv, D, FA2_DTYPE_FP16) || check_cache(batch, 1, page_size, table_width)) return 0;
  return decode_workspace_floats(batch, Hq, Hkv, D, table_width, page_size) * sizeof(float);
}

int fa2_decode(const void* q, const void* k_cache, const void* v_cache, void* out, const int* block_table,
               const int* lengths, void* workspace, size_t workspace_bytes, int batch, int Hq, int Hkv, int D, int pages,
               int page_size, int table_width, int dtype, float scale, const long long* strides, fa2_stream_t stream) {
  if (!q || !k_cache || !v_cache || !out || !block_table || !lengths) return FA2_ERR_NULL_POINTER;
  if (int e = check_heads(Hq, Hkv, D, dtype)) return e;
  if (int e = check_cache(batch, pages, page_size, table_width)) return e;
  // query heads of the call; the units of 64 keys that its CTAs share out
  if (static_cast<long long>(batch) * Hq > 0x7fffffffll ||
      (static_cast<long long>(table_width) * page_size / 64 + 3) * batch > 0x7fffffffll / Hkv)
    return FA2_ERR_SHAPE;
  for (const void* p : {q, k_cache, v_cache, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (!aligned_to(p, 16)) return FA2_ERR_MISALIGNED;
  if (!std::isfinite(scale) || !(scale > 0.f)) return FA2_ERR_SCALE;
  const size_t need = fa2_decode_workspace_bytes(batch, Hq, Hkv, D, page_size, table_width);
  if (need && (!workspace || workspace_bytes < need)) return FA2_ERR_WORKSPACE;
  DecodeArgs a{q, k_cache, v_cache, out, block_table, lengths, static_cast<float*>(workspace), row_strides(strides, Hq, D),
               cache_strides(strides ? strides + 2 : nullptr, page_size, Hkv, D),
               cache_strides(strides ? strides + 5 : nullptr, page_size, Hkv, D), strides ? strides[8] : table_width,
               batch, Hq, Hkv, D, pages, page_size, table_width, scale * 1.4426950408889634f};
  if (!rows_ok(a.sq, batch, Hq, D) || !cache_ok(a.sk_cache, pages, page_size, Hkv, D) ||
      !cache_ok(a.sv_cache, pages, page_size, Hkv, D) || (batch > 1 && a.table_stride < 0))
    return FA2_ERR_STRIDE;
  LaunchCtx ctx;
  if (int e = launch_context(&ctx)) return e;
  CUtensorMap tk, tv;
  const CacheStrides* const st[2] = {&a.sk_cache, &a.sv_cache};
  // A row is one head of one position; beside it stand other heads, which are read at another time, so the L2 must not fetch
  // more than the row.  Fetched 256 bytes at a time, rows of 128 bytes took twice as long (64 sequences of 230 000 keys, 12 heads of
  // 64 columns: 235 us).
  const CUtensorMapL2promotion promotion =
      D >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : (D >= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_NONE);
  for (int i = 0; i < 2; ++i) {
    // strides of dimensions of size 1 carry no information
    const long long slot = page_size > 1 ? st[i]->slot : D, head = Hkv > 1 ? st[i]->head : D, page = pages > 1 ? st[i]->page : D;
    if (int e = encode_map(i ? &tv : &tk, i ? v_cache : k_cache, dtype, pages, Hkv, page_size, D, Strides{page, head, slot}, 64,
                           decode_box_rows(page_size), CU_TENSOR_MAP_SWIZZLE_128B, promotion))
      return e;
  }
  return static_cast<int>(launch_decode(tk, tv, a, dtype, ctx.num_sms, ctx.status, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
