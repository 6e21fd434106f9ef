// Python entry of the paged-cache operators: argument checks, output
// allocation and the C-ABI call in one compiled step.
//
// A decode step calls these operators a few times per layer on a few tokens:
// the kernels take 3 us, and checking eleven tensors from Python and passing
// twenty arguments through ctypes takes 20.  Each function here serves a call
// whose tensors are as the kernels take them (types, layouts, one device) and
// returns None for any other, without having done anything; the Python
// wrappers in ops.py then convert or refuse.  The return code of the C entry
// comes back first, for ops.py to raise on.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/leanselect_b200.h"

namespace {

using at::Tensor;

// The tensor behind a Python argument; null when it is something else.
const Tensor* tensor_arg(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

// A contiguous tensor of this type on device `dev`.
bool plain(const Tensor* t, at::ScalarType type, int dev) {
  return t != nullptr && t->is_cuda() && t->get_device() == dev && t->scalar_type() == type &&
         t->is_contiguous() && !t->is_conj() && !t->is_neg();
}

bool vec(const Tensor* t, at::ScalarType type, int dev, int64_t n) {
  return plain(t, type, dev) && t->dim() == 1 && t->size(0) == n;
}

template <typename T>
T* ptr(const Tensor* t) {
  return t->numel() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// The cache's four tensors; fills pages, heads and head_dim.
bool cache_args(const Tensor* kp, const Tensor* vp, const Tensor* ks, const Tensor* vs, int dev,
                int64_t* pages, int64_t* heads, int64_t* dim) {
  if (!plain(kp, at::kFloat8_e4m3fn, dev) || !plain(vp, at::kFloat8_e4m3fn, dev) ||
      !plain(ks, at::kFloat, dev) || !plain(vs, at::kFloat, dev))
    return false;
  if (kp->dim() != 4 || kp->size(2) != LS_PAGE_TOKENS || !vp->sizes().equals(kp->sizes()) ||
      ks->dim() != 2 || !vs->sizes().equals(ks->sizes()) || ks->size(0) != kp->size(0) ||
      ks->size(1) != kp->size(1))
    return false;
  *pages = kp->size(0);
  *heads = kp->size(1);
  *dim = kp->size(3);
  return true;
}

// [N, G, D] bf16 with contiguous heads and 16-byte aligned tokens.
bool token_rows(const Tensor* t, int dev, int64_t g, int64_t d) {
  return t != nullptr && t->is_cuda() && t->get_device() == dev &&
         t->scalar_type() == at::kBFloat16 && t->dim() == 3 && t->size(1) == g &&
         t->size(2) == d && t->stride(2) == 1 && t->stride(1) == d && t->stride(0) % 8 == 0 &&
         t->stride(0) >= g * d && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
}

// Elements [from, from + n) of this type in a buffer, as a vector sharing its storage.
Tensor slice(const Tensor& buffer, at::ScalarType type, int64_t from, int64_t n) {
  auto impl = c10::make_intrusive<at::TensorImpl>(
      c10::Storage(buffer.storage()), buffer.key_set(), c10::scalarTypeToTypeMeta(type));
  impl->set_storage_offset(from);
  impl->set_sizes_contiguous({n});
  return Tensor(std::move(impl));
}

bool fits32(int64_t x) { return x >= 0 && x < (int64_t{1} << 31); }

// plan_pages(context_lens, new_lens, block_table, free_pages, free_head, total_new, status)
//   -> None | (code, seq_lens, cu_seqlens_q, cu_blocks, slots, positions, free_head)
PyObject* plan_pages(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7) Py_RETURN_NONE;
  const Tensor *ctx = tensor_arg(args[0]), *add = tensor_arg(args[1]), *table = tensor_arg(args[2]),
               *pool = tensor_arg(args[3]), *head = tensor_arg(args[4]),
               *status = tensor_arg(args[6]);
  if (ctx == nullptr || !ctx->is_cuda()) Py_RETURN_NONE;
  const int dev = ctx->get_device();
  const int64_t total = PyLong_AsLongLong(args[5]);
  if (total == -1 && PyErr_Occurred()) return nullptr;
  if (!plain(ctx, at::kInt, dev) || ctx->dim() != 1) Py_RETURN_NONE;
  const int64_t batch = ctx->size(0);
  if (batch < 1 || !fits32(batch) || !vec(add, at::kInt, dev, batch) ||
      !plain(table, at::kInt, dev) || table->dim() != 2 || table->size(0) != batch ||
      table->size(1) < 1 || !fits32(table->size(1)) || !plain(pool, at::kInt, dev) ||
      pool->dim() != 1 || !fits32(pool->size(0)) || !plain(head, at::kInt, dev) ||
      head->numel() != 1 || !vec(status, at::kInt, dev, 1) || !fits32(total))
    Py_RETURN_NONE;
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const auto opts = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(dev));
  // One allocation: slots, positions (each 16-byte aligned), then the int32 results.
  const int64_t even = (total + 1) / 2 * 2, ints = 4 * even;
  const Tensor buffer = at::empty({16 * even + 4 * (3 * batch + 3)}, opts.dtype(at::kByte));
  int64_t* l = static_cast<int64_t*>(buffer.data_ptr());
  int32_t* i = reinterpret_cast<int32_t*>(l + 2 * even);
  void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ls_plan_pages(ptr<int32_t>(ctx), ptr<int32_t>(add), static_cast<int32_t>(batch),
                     ptr<int32_t>(table), static_cast<int32_t>(table->size(1)), ptr<int32_t>(pool),
                     static_cast<int32_t>(pool->size(0)), ptr<int32_t>(head), total, i, i + batch,
                     i + 2 * batch + 1, l, l + even, i + 3 * batch + 2,
                     ptr<int32_t>(status), stream);
  Py_END_ALLOW_THREADS
  const auto vec32 = [&](int64_t from, int64_t n) {
    return THPVariable_Wrap(slice(buffer, at::kInt, ints + from, n));
  };
  return Py_BuildValue("(iNNNNNN)", rc, vec32(0, batch), vec32(batch, batch + 1),
                       vec32(2 * batch + 1, batch + 1),
                       THPVariable_Wrap(slice(buffer, at::kLong, 0, total)),
                       THPVariable_Wrap(slice(buffer, at::kLong, even, total)),
                       vec32(3 * batch + 2, 1));
  END_HANDLE_TH_ERRORS
}

// append_kv(k, v, context_lens, seq_lens, cu_seqlens_q, cu_blocks, slots, k_pages, v_pages,
//           k_scale, v_scale, status) -> None | code
PyObject* append_kv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 12) Py_RETURN_NONE;
  const Tensor* t[12];
  for (int i = 0; i < 12; ++i) t[i] = tensor_arg(args[i]);
  if (t[0] == nullptr || !t[0]->is_cuda() || t[2] == nullptr) Py_RETURN_NONE;
  const int dev = t[0]->get_device();
  int64_t pages, heads, dim;
  if (!cache_args(t[7], t[8], t[9], t[10], dev, &pages, &heads, &dim) ||
      !token_rows(t[0], dev, heads, dim) || !token_rows(t[1], dev, heads, dim))
    Py_RETURN_NONE;
  const int64_t n = t[0]->size(0), batch = t[2]->numel();
  if (n < 1 || t[1]->size(0) != n || !fits32(batch) || !fits32(heads) || !fits32(dim) ||
      !vec(t[2], at::kInt, dev, batch) || !vec(t[3], at::kInt, dev, batch) ||
      !vec(t[4], at::kInt, dev, batch + 1) || !vec(t[5], at::kInt, dev, batch + 1) ||
      !vec(t[6], at::kLong, dev, n) || !vec(t[11], at::kInt, dev, 1))
    Py_RETURN_NONE;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ls_append_kv(ptr<uint16_t>(t[0]), ptr<uint16_t>(t[1]), t[0]->stride(0), t[1]->stride(0), n,
                    static_cast<int32_t>(batch), static_cast<int32_t>(heads),
                    static_cast<int32_t>(dim), ptr<int32_t>(t[2]), ptr<int32_t>(t[3]),
                    ptr<int32_t>(t[4]), ptr<int32_t>(t[5]), ptr<int64_t>(t[6]), ptr<uint8_t>(t[7]),
                    ptr<uint8_t>(t[8]), ptr<float>(t[9]), ptr<float>(t[10]), pages,
                    ptr<int32_t>(t[11]), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// paged_attn(q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q,
//            max_seqlen_q, max_seqlen_k, topk_idx, scale, causal, return_lse, out, status)
//   -> None | (code, out, lse or None)
PyObject* paged_attn(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 16) Py_RETURN_NONE;
  const Tensor* t[8];
  for (int i = 0; i < 8; ++i) t[i] = tensor_arg(args[i]);
  const Tensor* q = t[0];
  if (q == nullptr || !q->is_cuda()) Py_RETURN_NONE;
  const int dev = q->get_device();
  int64_t pages, heads, dim;
  if (!cache_args(t[1], t[2], t[3], t[4], dev, &pages, &heads, &dim) ||
      !plain(q, at::kBFloat16, dev) || q->dim() != 3 || q->size(2) != dim || heads < 1 ||
      q->size(1) % heads != 0)
    Py_RETURN_NONE;
  const int64_t n = q->size(0), h = q->size(1);
  const Tensor *table = t[5], *seq = t[6];
  if (!plain(table, at::kInt, dev) || table->dim() != 2 || !plain(seq, at::kInt, dev) ||
      seq->dim() != 1)
    Py_RETURN_NONE;
  const int64_t batch = seq->size(0);
  if (table->size(0) != batch || !vec(t[7], at::kInt, dev, batch + 1) || !fits32(batch) ||
      !fits32(table->size(1)) || !fits32(h) || !fits32(heads) || !fits32(dim))
    Py_RETURN_NONE;
  const int64_t max_q = PyLong_AsLongLong(args[8]), max_k = PyLong_AsLongLong(args[9]);
  const double scale = PyFloat_AsDouble(args[11]);
  if (PyErr_Occurred()) return nullptr;
  if (!fits32(max_q) || !fits32(max_k)) Py_RETURN_NONE;
  const Tensor* idx = nullptr;
  if (args[10] != Py_None) {
    idx = tensor_arg(args[10]);
    if (!plain(idx, at::kInt, dev) || idx->dim() != 3 || idx->size(0) != heads ||
        idx->size(1) != n || idx->size(2) < 1 || !fits32(idx->size(2)))
      Py_RETURN_NONE;
  }
  const Tensor *given = nullptr, *status = tensor_arg(args[15]);
  if (args[14] != Py_None) {
    given = tensor_arg(args[14]);
    if (!plain(given, at::kBFloat16, dev) || !given->sizes().equals(q->sizes())) Py_RETURN_NONE;
  }
  if (!vec(status, at::kInt, dev, 1)) Py_RETURN_NONE;
  const bool causal = args[12] == Py_True, want_lse = args[13] == Py_True;
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  const auto opts = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(dev));
  const Tensor out = given ? *given : at::empty(q->sizes(), opts.dtype(at::kBFloat16));
  Tensor lse;
  if (want_lse) lse = at::empty({h, n}, opts.dtype(at::kFloat));
  const int64_t bytes = static_cast<int64_t>(ls_paged_attn_workspace_bytes());
  const Tensor ws = at::empty({bytes}, opts.dtype(at::kByte));
  void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ls_paged_attn(ptr<uint16_t>(q), ptr<uint8_t>(t[1]), ptr<uint8_t>(t[2]), ptr<float>(t[3]),
                     ptr<float>(t[4]), pages, ptr<int32_t>(table),
                     static_cast<int32_t>(table->size(1)), ptr<int32_t>(seq), ptr<int32_t>(t[7]),
                     static_cast<int32_t>(batch), static_cast<int32_t>(max_q),
                     static_cast<int32_t>(max_k), n, static_cast<int32_t>(h),
                     static_cast<int32_t>(heads), static_cast<int32_t>(dim),
                     idx ? ptr<int32_t>(idx) : nullptr,
                     idx ? static_cast<int32_t>(idx->size(2)) : 0, static_cast<float>(scale),
                     causal ? 1 : 0, ws.data_ptr(), static_cast<size_t>(bytes), ptr<uint16_t>(&out),
                     want_lse && n ? lse.data_ptr<float>() : nullptr, ptr<int32_t>(status), stream);
  Py_END_ALLOW_THREADS
  PyObject* lse_obj = Py_None;
  if (want_lse) lse_obj = THPVariable_Wrap(lse); else Py_INCREF(lse_obj);
  return Py_BuildValue("(iNN)", rc, THPVariable_Wrap(out), lse_obj);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"plan_pages", reinterpret_cast<PyCFunction>(plan_pages), METH_FASTCALL, nullptr},
    {"append_kv", reinterpret_cast<PyCFunction>(append_kv), METH_FASTCALL, nullptr},
    {"paged_attn", reinterpret_cast<PyCFunction>(paged_attn), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&kModule); }
