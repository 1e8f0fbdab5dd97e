// Host path of attention over packed sequences, forward and backward, as a C++ autograd function.
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>

#include "host.h"

namespace fa2_host {
namespace {

struct Sizes {
  int rows, batch, Hq, Hkv, D;
};

// q, k, v, (dout,) each [rows, heads, D]
template <size_t N>
std::array<long long, 2 * N> strides_of(const std::array<const at::Tensor*, N>& ts) {
  std::array<long long, 2 * N> s;
  for (size_t i = 0; i < N; ++i) s[2 * i] = ts[i]->stride(0), s[2 * i + 1] = ts[i]->stride(1);
  return s;
}
at::Tensor dense_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); }
at::Tensor bytes_on(const at::Tensor& t, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, t.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
}
cudaStream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The plan and, behind it, lse in one allocation.
size_t lse_offset(const Sizes& n) { return fa2_packed_plan_bytes(n.rows, n.batch); }
size_t scratch_bytes(const Sizes& n) { return lse_offset(n) + 4ull * n.Hq * n.rows; }
float* lse_of(const at::Tensor& scratch, const Sizes& n) {
  return reinterpret_cast<float*>(static_cast<char*>(scratch.data_ptr()) + lse_offset(n));
}

struct Forward {
  at::Tensor out, scratch;
};
// q, k and v are replaced by what the kernels read.
Forward run_forward(at::Tensor& q, at::Tensor& k, at::Tensor& v, const at::Tensor& cu, const Sizes& n, double scale) {
  const c10::cuda::CUDAGuard guard(q.device());
  q = rows_input(q), k = rows_input(k), v = rows_input(v);
  Forward r{dense_like(q), bytes_on(q, scratch_bytes(n))};
  if (n.rows == 0) return r;
  const auto strides = strides_of<3>({&q, &k, &v});
  check_code("fa2_packed_fwd", fa2_packed_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), r.out.data_ptr(), lse_of(r.scratch, n),
                                              cu.data_ptr<int>(), r.scratch.data_ptr(), n.rows, n.batch, n.Hq, n.Hkv, n.D, dtype_code(q),
                                              static_cast<float>(scale), strides.data(), stream_of(q)));
  return r;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  // `r` holds the outputs of the forward kernel, already launched on saved q, k and v.
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const std::array<at::Tensor, 3>& saved, const at::Tensor& cu, const Forward& r, double scale) {
    ctx->save_for_backward({saved[0], saved[1], saved[2], cu, r.out, r.scratch});
    ctx->saved_data["scale"] = scale;
    return r.out.view(r.out.sizes());  // the tensor that is saved is not the one handed out
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!c10::GradMode::is_enabled(), "flash_attention_packed has no second derivative: do not pass create_graph=True");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &cu = saved[3], &out = saved[4], &scratch = saved[5];
    // saved-tensor hooks must give back what was saved
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && out.sizes() == q.sizes() && k.size(0) == q.size(0) &&
                    k.size(2) == q.size(2) && cu.dim() == 1 && cu.size(0) > 1 && k.size(1) > 0 && q.size(1) % k.size(1) == 0,
                "the saved tensors have changed their shapes");
    for (const at::Tensor* t : {&q, &k, &v, &out})
      TORCH_CHECK(is_16bit(*t) && t->scalar_type() == q.scalar_type() && rows_readable(*t), "the saved tensors have changed their type or strides");
    const Sizes n{static_cast<int>(q.size(0)), static_cast<int>(cu.size(0)) - 1, static_cast<int>(q.size(1)), static_cast<int>(k.size(1)),
                  static_cast<int>(q.size(2))};
    TORCH_CHECK(out.is_contiguous() && cu.is_contiguous() && cu.scalar_type() == at::kInt && scratch.is_contiguous() &&
                    scratch.nbytes() == scratch_bytes(n) && reinterpret_cast<uintptr_t>(scratch.data_ptr()) % 16 == 0,
                "the saved tensors have changed their type or strides");
    at::Tensor dout = grads[0];
    TORCH_CHECK(dout.sizes() == q.sizes(), "the gradient must have the shape of the output");
    for (const at::Tensor* t : {&q, &k, &v, &cu, &out, &scratch, static_cast<const at::Tensor*>(&dout)})
      TORCH_CHECK(t->is_cuda() && t->device() == q.device(), "the saved tensors or the gradient are on another device");
    const c10::cuda::CUDAGuard guard(q.device());
    if (dout.scalar_type() != q.scalar_type()) dout = dout.to(q.scalar_type());
    dout = rows_input(dout.is_neg() ? dout.resolve_neg() : dout);
    at::Tensor dq = dense_like(q), dk = dense_like(k), dv = dense_like(v);
    if (n.rows > 0) {
      const size_t bytes = fa2_packed_bwd_workspace_bytes(n.rows, n.batch, n.Hq);
      const at::Tensor workspace = bytes_on(q, bytes);
      const auto strides = strides_of<4>({&q, &k, &v, &dout});
      check_code("fa2_packed_bwd",
                 fa2_packed_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse_of(scratch, n), dq.data_ptr(),
                                dk.data_ptr(), dv.data_ptr(), cu.data_ptr<int>(), scratch.data_ptr(), workspace.data_ptr(), bytes, n.rows,
                                n.batch, n.Hq, n.Hkv, n.D, dtype_code(q), static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                strides.data(), stream_of(q)));
    }
    {
      pybind11::gil_scoped_acquire gil;
      check_status_if_asked("fa2_packed_bwd", q);
    }
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

// packed(q, k, v, cu_seqlens, scale or None) -> output
PyObject* packed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) return PyErr_Format(PyExc_TypeError, "packed takes 5 arguments");
  const at::Tensor q = tensor_argument(args[0], "q"), k = tensor_argument(args[1], "k"), v = tensor_argument(args[2], "v");
  const at::Tensor cu = tensor_argument(args[3], "cu_seqlens");
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                    "q must be [tokens, heads, headdim], k and v [tokens, kv_heads, headdim]");
  const int64_t d = q.size(2);
  TORCH_CHECK_VALUE(d >= 8 && d <= 128 && d % 8 == 0, "head dimension ", std::to_string(d), " is not supported (multiples of 8 up to 128)");
  TORCH_CHECK_VALUE(q.size(1) > 0 && q.size(1) <= 65535 && k.size(1) > 0 && q.size(1) % k.size(1) == 0, "heads must be a multiple of kv_heads");
  TORCH_CHECK_VALUE(is_16bit(q) && q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k and v must be fp16 or bf16, all the same");
  check_int32(cu, "cu_seqlens", 1);
  TORCH_CHECK_VALUE(cu.size(0) >= 2 && cu.size(0) <= (1 << 20) + 1, "cu_seqlens must have one entry more than there are sequences");
  TORCH_CHECK_VALUE(q.size(0) <= (1 << 24), "too many tokens");
  const double scale = scale_argument(args[4], d);
  TORCH_CHECK_VALUE(std::isfinite(scale) && scale > 0, "softmax scale must be finite and > 0");
  check_devices({{&q, "q"}, {&k, "k"}, {&v, "v"}, {&cu, "cu_seqlens"}});
  const Sizes n{static_cast<int>(q.size(0)), static_cast<int>(cu.size(0)) - 1, static_cast<int>(q.size(1)), static_cast<int>(k.size(1)),
                static_cast<int>(d)};
  at::Tensor result;
  {
    pybind11::gil_scoped_release no_gil;
    std::array<at::Tensor, 3> in{q, k, v};
    Forward r;
    {
      const at::AutoGradMode no_grad(false);
      r = run_forward(in[0], in[1], in[2], cu, n, scale);
    }
    const bool graph = c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    result = graph ? PackedAttention::apply(q, k, v, in, cu, r, scale) : r.out;
  }
  check_status_if_asked("fa2_packed_fwd", q);
  return THPVariable_Wrap(result);
  END_HANDLE_TH_ERRORS
}

}  // namespace fa2_host
