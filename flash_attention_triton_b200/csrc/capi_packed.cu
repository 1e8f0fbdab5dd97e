// C entry points of attention over packed sequences: argument checks, tensor maps and launches.
#include <cmath>

#include "../../include/fa2_b200.h"
#include "capi.cuh"
#include "packed.cuh"

namespace fa2 {
namespace {

int check_packed(int rows, int batch, int Hq, int Hkv, int D, int dtype, float scale) {
  if (int e = check_heads(Hq, Hkv, D, dtype)) return e;
  if (D > 128) return FA2_ERR_HEAD_DIM;
  if (rows < 0 || rows > (1 << 24) || batch < 1 || batch > (1 << 20)) return FA2_ERR_SHAPE;
  // CTAs of the backward, and the numbers that the forward's CTAs draw
  if (4ll * packed_capacity(rows, batch) * (Hq + 8) + 1024 > 0x7fffffffll) return FA2_ERR_SHAPE;
  return std::isfinite(scale) && scale > 0.f ? FA2_OK : FA2_ERR_SCALE;
}

// A [rows, H, D] tensor; strides == NULL: dense.
struct Rows {
  const void* p;
  int H;
  RowStrides st;
  Rows(const void* base, int heads, int D, const long long* strides)
      : p(base), H(heads), st{strides ? strides[0] : static_cast<long long>(heads) * D, strides ? strides[1] : D} {}
  bool ok(int rows, int D) const { return stride_ok(st.row, rows, D) && stride_ok(st.head, H, D); }
  int map(CUtensorMap* m, int rows, int D, int dtype, int box_rows) const {
    // strides of dimensions of size 1 carry no information
    const long long head = H > 1 ? st.head : D, row = rows > 1 ? st.row : static_cast<long long>(H) * D;
    return make_map(m, p, dtype, 1, H, rows, D, Strides{row, head, row}, box_rows);
  }
};

PackedShape make_shape(int rows, int batch, int Hq, int Hkv, int D, int dtype, float scale) {
  return PackedShape{rows, batch, Hq, Hkv, padded_head_dim(D), D, dtype, scale};
}

}  // namespace
}  // namespace fa2

using namespace fa2;

extern "C" {

size_t fa2_packed_plan_bytes(int rows, int batch) {
  return rows < 0 || rows > (1 << 24) || batch < 1 || batch > (1 << 20) ? 0 : packed_plan_bytes(rows, batch);
}

int fa2_packed_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* cu_seqlens, void* plan,
                   int rows, int batch, int Hq, int Hkv, int D, int dtype, float scale, const long long* strides,
                   fa2_stream_t stream) {
  if (!q || !k || !v || !o || !lse || !cu_seqlens || !plan) return FA2_ERR_NULL_POINTER;
  if (int e = check_packed(rows, batch, Hq, Hkv, D, dtype, scale)) return e;
  for (const void* p : {q, k, v, static_cast<const void*>(o), static_cast<const void*>(plan)})
    if (!aligned_to(p, 16)) return FA2_ERR_MISALIGNED;
  const Rows tq_(q, Hq, D, strides), tk_(k, Hkv, D, strides ? strides + 2 : nullptr), tv_(v, Hkv, D, strides ? strides + 4 : nullptr),
      to_(o, Hq, D, nullptr);
  for (const Rows* t : {&tq_, &tk_, &tv_})
    if (!t->ok(rows, D)) return FA2_ERR_STRIDE;
  if (rows == 0) return FA2_OK;
  LaunchCtx ctx;
  if (int e = launch_context(&ctx)) return e;
  CUtensorMap tq, tk, tv, to;
  if (int e = tq_.map(&tq, rows, D, dtype, 128)) return e;
  if (int e = tk_.map(&tk, rows, D, dtype, 128)) return e;
  if (int e = tv_.map(&tv, rows, D, dtype, 128)) return e;
  if (int e = to_.map(&to, rows, D, dtype, 32)) return e;
  const PackedShape s = make_shape(rows, batch, Hq, Hkv, D, dtype, scale);
  const PackedPlan p = packed_plan(plan, rows, batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!packed_fwd_alone(s, ctx.num_sms))
    if (cudaError_t e = launch_packed_plan(s, cu_seqlens, p, Hq / Hkv % 2 != 0, o, ctx.status, ctx.num_sms, st)) return static_cast<int>(e);
  return static_cast<int>(launch_packed_fwd(s, cu_seqlens, p, tq, tk, tv, to, o, lse, ctx.status, ctx.num_sms, st));
}

size_t fa2_packed_bwd_workspace_bytes(int rows, int batch, int Hq) {
  return rows < 0 || rows > (1 << 24) || batch < 1 || batch > (1 << 20) || Hq < 1 ? 0 : packed_stats_bytes(rows, batch, Hq);
}

int fa2_packed_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse, void* dq,
                   void* dk, void* dv, const int* cu_seqlens, const void* plan, void* workspace, size_t workspace_bytes,
                   int rows, int batch, int Hq, int Hkv, int D, int dtype, float scale, const long long* strides,
                   fa2_stream_t stream) {
  if (!q || !k || !v || !o || !dout || !lse || !dq || !dk || !dv || !cu_seqlens || !plan) return FA2_ERR_NULL_POINTER;
  if (int e = check_packed(rows, batch, Hq, Hkv, D, dtype, scale)) return e;
  for (const void* p : {q, k, v, o, dout, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv),
                        plan, static_cast<const void*>(workspace)})
    if (!aligned_to(p, 16)) return FA2_ERR_MISALIGNED;
  const Rows tq_(q, Hq, D, strides), tk_(k, Hkv, D, strides ? strides + 2 : nullptr), tv_(v, Hkv, D, strides ? strides + 4 : nullptr),
      tdo_(dout, Hq, D, strides ? strides + 6 : nullptr), tdq_(dq, Hq, D, nullptr), tdk_(dk, Hkv, D, nullptr), tdv_(dv, Hkv, D, nullptr);
  for (const Rows* t : {&tq_, &tk_, &tv_, &tdo_})
    if (!t->ok(rows, D)) return FA2_ERR_STRIDE;
  if (rows == 0) return FA2_OK;
  if (!workspace || workspace_bytes < packed_stats_bytes(rows, batch, Hq)) return FA2_ERR_WORKSPACE;
  LaunchCtx ctx;
  if (int e = launch_context(&ctx)) return e;
  const PackedShape s = make_shape(rows, batch, Hq, Hkv, D, dtype, scale);
  const PackedPlan p = packed_plan(const_cast<void*>(plan), rows, batch);
  unsigned* const words = static_cast<unsigned*>(workspace);
  const size_t heads = static_cast<size_t>(p.capacity) * Hq;
  const PackedStats stats{static_cast<float*>(workspace), words + heads * 256, words + heads * (256 + 4)};
  const int cluster = packed_cluster(s, ctx.num_sms);
  const int step = cluster > 1 ? 128 : packed_step_rows(s, Hkv, ctx.num_sms), dq_step = packed_step_rows(s, Hq, ctx.num_sms);
  CUtensorMap tq, tk, tv, tdo, tdq, tdk, tdv;
  if (int e = tq_.map(&tq, rows, D, dtype, step)) return e;
  if (int e = tdo_.map(&tdo, rows, D, dtype, step)) return e;
  if (int e = tk_.map(&tk, rows, D, dtype, 128)) return e;
  if (int e = tv_.map(&tv, rows, D, dtype, 128)) return e;
  if (int e = tdq_.map(&tdq, rows, D, dtype, 32)) return e;
  if (int e = tdk_.map(&tdk, rows, D, dtype, 32)) return e;
  if (int e = tdv_.map(&tdv, rows, D, dtype, 32)) return e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cudaError_t e = launch_packed_preprocess(s, p, cu_seqlens, o, dout, tdo_.st, lse, stats, dq, dk, dv, st)) return static_cast<int>(e);
  if (cudaError_t e = launch_packed_dkdv(s, p, tq, tk, tv, tdo, tdk, tdv, dk, dv, stats, step, cluster, ctx.status, st)) return static_cast<int>(e);
  // the other kernel holds Q and dO and walks K and V
  if (step != 128) {
    if (int e = tq_.map(&tq, rows, D, dtype, 128)) return e;
    if (int e = tdo_.map(&tdo, rows, D, dtype, 128)) return e;
  }
  if (dq_step != 128) {
    if (int e = tk_.map(&tk, rows, D, dtype, dq_step)) return e;
    if (int e = tv_.map(&tv, rows, D, dtype, dq_step)) return e;
  }
  return static_cast<int>(launch_packed_dq(s, p, tq, tk, tv, tdo, tdq, dq, stats, dq_step, ctx.status, st));
}

}  // extern "C"
