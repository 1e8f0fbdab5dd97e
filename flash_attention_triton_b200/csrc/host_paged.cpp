// Host path of the paged key-value cache: checks, allocation, strides, current stream, device guard, the C ABI calls.
#include "host.h"

namespace fa2_host {

bool rows_readable(const at::Tensor& t) {
  if ((t.size(2) > 1 && t.stride(2) != 1) || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int i = 0; i < 2; ++i)
    if (t.size(i) > 1 && (t.stride(i) < t.size(2) || t.stride(i) % 8)) return false;
  return true;
}

void check_int32(const at::Tensor& t, const char* name, int dims) {
  TORCH_CHECK_VALUE(t.dim() == dims && t.scalar_type() == at::kInt, name, dims == 1 ? " must be an int32 tensor of one dimension" : " must be an int32 tensor of two dimensions");
  TORCH_CHECK_VALUE(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, name, " must be contiguous in its last dimension");
}

void check_devices(std::initializer_list<std::pair<const at::Tensor*, const char*>> tensors) {
  const at::Tensor* first = nullptr;
  for (const auto& [t, name] : tensors) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) {
      pybind11::gil_scoped_acquire gil;
      PyErr_SetString(PyExc_AssertionError, "All tensors must reside on CUDA device");
      throw python_error();
    }
    if (!first) first = t;
    TORCH_CHECK_VALUE(t->device() == first->device(), name, " is on another device than the other tensors");
  }
}

namespace {

struct Cache {
  int batch, pages, page_size, table_width, Hkv, D;
};

// k_cache and v_cache [pages, page_size, Hkv, D], block_table [batch, width], lengths [batch]
Cache check_cache(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths) {
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(),
                    "k_cache and v_cache must be [pages, page_size, kv_heads, headdim] tensors of the same shape");
  TORCH_CHECK_VALUE(is_16bit(k_cache) && k_cache.scalar_type() == v_cache.scalar_type(), "k_cache and v_cache must be fp16 or bf16, both the same");
  const int64_t d = k_cache.size(3);
  TORCH_CHECK_VALUE(d >= 8 && d <= 256 && d % 8 == 0, "head dimension ", std::to_string(d), " is not supported (multiples of 8 up to 256)");
  TORCH_CHECK_VALUE(k_cache.size(0) > 0 && k_cache.size(1) > 0 && k_cache.size(2) > 0, "the cache has no pages, slots or heads");
  for (const at::Tensor* t : {&k_cache, &v_cache}) {
    bool ok = t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t->size(i) == 1 || (t->stride(i) >= d && t->stride(i) % 8 == 0));
    TORCH_CHECK_VALUE(ok, "the cache must be 16-byte aligned, contiguous in its last dimension, with other strides that are multiples of 8");
  }
  check_int32(table, "block_table", 2);
  check_int32(lengths, "lengths", 1);
  TORCH_CHECK_VALUE(lengths.size(0) == table.size(0), "lengths and block_table must have one entry for each sequence");
  TORCH_CHECK_VALUE(table.size(0) > 0 && table.size(1) > 0, "block_table has no entries");
  TORCH_CHECK_VALUE(k_cache.size(0) <= INT32_MAX && table.size(0) <= (1 << 20) && table.size(1) <= INT32_MAX / k_cache.size(1),
                    "the cache or the block table is too large");
  return Cache{static_cast<int>(table.size(0)), static_cast<int>(k_cache.size(0)), static_cast<int>(k_cache.size(1)),
               static_cast<int>(table.size(1)), static_cast<int>(k_cache.size(2)), static_cast<int>(d)};
}

void check_no_graph(std::initializer_list<const at::Tensor*> tensors, const char* fn) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : tensors)
    TORCH_CHECK_VALUE(!t->defined() || !t->requires_grad(), fn, " has no gradient: call it under torch.no_grad()");
}

void put_rows(long long*& s, const at::Tensor& t) { *s++ = t.stride(0), *s++ = t.stride(1); }
void put_cache(long long*& s, const at::Tensor& t) { *s++ = t.stride(0), *s++ = t.stride(1), *s++ = t.stride(2); }

}  // namespace

// kv_append(k, v, k_cache, v_cache, block_table, lengths, cu_seqlens, q, cos, sin, interleaved, return_k)
//   -> (rotated q or None, rotated k or None)
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 12) return PyErr_Format(PyExc_TypeError, "kv_append takes 12 arguments");
  at::Tensor k = tensor_argument(args[0], "k"), v = tensor_argument(args[1], "v");
  const at::Tensor k_cache = written_argument(args[2], "k_cache"), v_cache = written_argument(args[3], "v_cache");
  const at::Tensor table = tensor_argument(args[4], "block_table"), lengths = tensor_argument(args[5], "lengths");
  const at::Tensor cu_seqlens = tensor_argument(args[6], "cu_seqlens", true);
  at::Tensor q = tensor_argument(args[7], "q", true);
  const at::Tensor cos = tensor_argument(args[8], "cos", true), sin = tensor_argument(args[9], "sin", true);
  const int interleaved = PyObject_IsTrue(args[10]), return_k = PyObject_IsTrue(args[11]);
  if (interleaved < 0 || return_k < 0) return nullptr;

  const Cache c = check_cache(k_cache, v_cache, table, lengths);
  TORCH_CHECK_VALUE(k.dim() == 3 && k.sizes() == v.sizes() && k.size(1) == c.Hkv && k.size(2) == c.D,
                    "k and v must be [tokens, kv_heads, headdim] tensors with the heads of the cache");
  const int64_t tokens = k.size(0);
  TORCH_CHECK_VALUE(tokens <= (1 << 24), "too many tokens");
  TORCH_CHECK_VALUE(k.scalar_type() == k_cache.scalar_type() && v.scalar_type() == k.scalar_type(), "k and v must have the type of the cache");
  if (q.defined()) {
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == tokens && q.size(2) == c.D && q.size(1) > 0 && q.size(1) <= 65535 && q.size(1) % c.Hkv == 0,
                      "q must be a [tokens, heads, headdim] tensor with a multiple of the cache's heads");
    TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type(), "q must have the type of the cache");
  }
  if (cu_seqlens.defined()) {
    check_int32(cu_seqlens, "cu_seqlens", 1);
    TORCH_CHECK_VALUE(cu_seqlens.size(0) == c.batch + 1, "cu_seqlens must have one entry more than there are sequences");
  } else {
    TORCH_CHECK_VALUE(tokens == c.batch, "without cu_seqlens there must be one token for each sequence");
  }
  TORCH_CHECK_VALUE(cos.defined() == sin.defined(), "cos and sin go together");
  int rotary = 0, positions = 0;
  if (cos.defined()) {
    TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat &&
                          cos.is_contiguous() && sin.is_contiguous() && cos.size(0) > 0 && cos.size(0) <= INT32_MAX,
                      "cos and sin must be contiguous fp32 [positions, rotated columns / 2] tensors");
    TORCH_CHECK_VALUE(cos.size(1) % 8 == 0 && cos.size(1) > 0 && 2 * cos.size(1) <= c.D, "the rotated columns must be a multiple of 16 up to the head dimension");
    TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(cos.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(sin.data_ptr()) % 16 == 0, "cos and sin must be 16-byte aligned");
    rotary = 2 * static_cast<int>(cos.size(1)), positions = static_cast<int>(cos.size(0));
  }
  check_no_graph({&k, &v, &q, &k_cache, &v_cache, &cos, &sin}, "append_kv_cache");
  check_devices({{&k, "k"}, {&v, "v"}, {&k_cache, "k_cache"}, {&v_cache, "v_cache"}, {&table, "block_table"},
                 {&lengths, "lengths"}, {&cu_seqlens, "cu_seqlens"}, {&q, "q"}, {&cos, "cos"}, {&sin, "sin"}});
  at::Tensor q_out, k_out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(k.device());
    k = rows_input(k), v = rows_input(v);
    if (q.defined()) {
      q = rows_input(q);
      q_out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    }
    if (return_k) k_out = at::empty(k.sizes(), k.options().memory_format(at::MemoryFormat::Contiguous));
    long long strides[13], *s = strides;
    put_rows(s, q.defined() ? q : k), put_rows(s, k), put_rows(s, v), put_cache(s, k_cache), put_cache(s, v_cache);
    *s = table.stride(0);
    if (tokens > 0)  // an empty tensor has no address
      check_code("fa2_kv_append",
               fa2_kv_append(q.defined() ? q.data_ptr() : nullptr, k.data_ptr(), v.data_ptr(), q.defined() ? q_out.data_ptr() : nullptr,
                             return_k ? k_out.data_ptr() : nullptr, k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr<int>(),
                             lengths.data_ptr<int>(), cu_seqlens.defined() ? cu_seqlens.data_ptr<int>() : nullptr,
                             rotary ? cos.data_ptr<float>() : nullptr, rotary ? sin.data_ptr<float>() : nullptr, static_cast<int>(tokens),
                             c.batch, q.defined() ? static_cast<int>(q.size(1)) : c.Hkv, c.Hkv, c.D, c.pages, c.page_size, c.table_width,
                             positions, rotary, interleaved, dtype_code(k), strides,
                             c10::cuda::getCurrentCUDAStream(k.device().index()).stream()));
    for (const at::Tensor* t : {&k_cache, &v_cache})  // autograd sees that they have been written
      if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  check_status_if_asked("fa2_kv_append", k);
  return Py_BuildValue("NN", THPVariable_Wrap(q_out), THPVariable_Wrap(k_out));
  END_HANDLE_TH_ERRORS
}

// decode(q, k_cache, v_cache, block_table, lengths, scale or None) -> output
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6) return PyErr_Format(PyExc_TypeError, "decode takes 6 arguments");
  at::Tensor q = tensor_argument(args[0], "q");
  const at::Tensor k_cache = tensor_argument(args[1], "k_cache"), v_cache = tensor_argument(args[2], "v_cache");
  const at::Tensor table = tensor_argument(args[3], "block_table"), lengths = tensor_argument(args[4], "lengths");
  const Cache c = check_cache(k_cache, v_cache, table, lengths);
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == c.batch && q.size(2) == c.D, "q must be a [batch, heads, headdim] tensor, one row for each sequence");
  TORCH_CHECK_VALUE(q.size(1) > 0 && q.size(1) <= 65535 && q.size(1) % c.Hkv == 0, "the heads of q must be a multiple of the cache's heads");
  TORCH_CHECK_VALUE(q.scalar_type() == k_cache.scalar_type(), "q must have the type of the cache");
  const double scale = scale_argument(args[5], c.D);
  check_no_graph({&q, &k_cache, &v_cache}, "flash_attention_decode");
  check_devices({{&q, "q"}, {&k_cache, "k_cache"}, {&v_cache, "v_cache"}, {&table, "block_table"}, {&lengths, "lengths"}});
  at::Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(q.device());
    q = rows_input(q);
    out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    const int Hq = static_cast<int>(q.size(1));
    const size_t bytes = fa2_decode_workspace_bytes(c.batch, Hq, c.Hkv, c.D, c.page_size, c.table_width);
    const at::Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
    long long strides[9], *s = strides;
    put_rows(s, q), put_cache(s, k_cache), put_cache(s, v_cache);
    *s = table.stride(0);
    check_code("fa2_decode", fa2_decode(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), table.data_ptr<int>(),
                                        lengths.data_ptr<int>(), workspace.data_ptr(), bytes, c.batch, Hq, c.Hkv, c.D, c.pages,
                                        c.page_size, c.table_width, dtype_code(q), static_cast<float>(scale), strides,
                                        c10::cuda::getCurrentCUDAStream(q.device().index()).stream()));
  }
  check_status_if_asked("fa2_decode", q);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace fa2_host
