// Host path of the paged serving calls: tensors in, C ABI calls (include/hfan.h)
// out.  A decode step makes these calls in every layer, for kernels of a few
// microseconds, and descriptors, views, allocations and the call itself cost
// about 20 us through ctypes; here they cost about 5.  Nothing else of the
// package needs torch's C++ interface.
//
// Arguments arrive positionally from ops.py, which has checked shapes, types and
// devices.  The entry points are those of the library that the package has
// loaded (bind()).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/hfan.h"

namespace {

decltype(&hfan_paged_append) fn_append;
decltype(&hfan_paged_chunk_workspace_bytes) fn_bytes;
decltype(&hfan_paged_chunk_fwd) fn_chunk;
decltype(&hfan_paged_evict) fn_evict;
decltype(&hfan_last_error) fn_error;

struct PyFailure {};  // a Python exception is set

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "a tensor was expected");
    throw PyFailure();
  }
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailure();
  return v;
}
int32_t int32(PyObject* o) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) {
    PyErr_SetString(PyExc_ValueError, "a size does not fit in 32 bits");
    throw PyFailure();
  }
  return (int32_t)v;
}
int32_t size32(int64_t v) {
  if (v > INT32_MAX) {
    PyErr_SetString(PyExc_ValueError, "a size does not fit in 32 bits");
    throw PyFailure();
  }
  return (int32_t)v;
}

// 64-bit integers saturate: cut to 32 bits, a wild length or page id could pass
// for a valid one, which the kernels then would not record.
at::Tensor ints(const at::Tensor& t) {
  if (t.scalar_type() == at::kInt) return t.contiguous();
  return t.clamp(at::Scalar(INT32_MIN), at::Scalar(INT32_MAX)).to(at::kInt).contiguous();
}
at::Tensor rows(const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }
hfan_tensor view(const at::Tensor& t) { return hfan_tensor{t.data_ptr(), 0, t.stride(1), t.stride(0)}; }

int32_t dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return HFAN_FLOAT32;
    case at::kHalf: return HFAN_FLOAT16;
    case at::kBFloat16: return HFAN_BFLOAT16;
    default:
      PyErr_Format(PyExc_ValueError, "unsupported dtype torch.%s; expected float32, float16 or bfloat16",
                   c10::toString(t.scalar_type()));
      throw PyFailure();
  }
}

void check(int rc, const char* what) {
  if (rc == HFAN_OK) return;
  if (rc == HFAN_ERR_INVALID)
    PyErr_SetString(PyExc_ValueError, fn_error());
  else
    PyErr_Format(PyExc_RuntimeError, "%s failed (status %d): %s", what, rc, fn_error());
  throw PyFailure();
}

// Runs body with C++ exceptions turned into Python ones.
template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& body) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments were expected, %zd given", want, n);
    return nullptr;
  }
  try {
    return body();
  } catch (const PyFailure&) {
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const c10::OutOfMemoryError& e) {
    // what torch itself raises, so that callers may catch torch.cuda.OutOfMemoryError
    PyObject* type = nullptr;
    if (PyObject* torch = PyImport_ImportModule("torch")) {
      type = PyObject_GetAttrString(torch, "OutOfMemoryError");
      Py_DECREF(torch);
    }
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

struct Weights {
  float* data = nullptr;
  int64_t ld = 0;
  explicit Weights(PyObject* o) {
    if (o == Py_None) return;
    const at::Tensor& t = tensor(o);
    data = t.data_ptr<float>();
    ld = t.stride(0);
  }
};

// A tensor that the kernels wrote in place: autograd finds out by its version
// when it had saved it.  (Inference tensors have none.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject* weights) {
  if (weights != Py_None) written(tensor(weights));
}

// (key, value, key_cache, value_cache, block_table, cu_seqlens, lengths, page_size, max_q, key_weights)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const at::Tensor key = rows(tensor(a[0])), value = rows(tensor(a[1]));
    const at::Tensor &kc = tensor(a[2]), &vc = tensor(a[3]);
    const c10::cuda::CUDAGuard guard(key.device());
    const at::Tensor table = ints(tensor(a[4])), cu = ints(tensor(a[5])), lens = ints(tensor(a[6]));
    const Weights w(a[9]);
    hfan_chunk_desc d{};
    d.dtype = dtype_of(key);
    d.normalizer = HFAN_SOFTMAX1;
    d.batch = size32(table.size(0));
    d.heads_q = d.heads_kv = size32(key.size(1));
    d.head_dim = size32(key.size(2));
    d.total_q = size32(key.size(0));
    d.max_len_q = int32(a[8]);
    d.page_size = int32(a[7]);
    d.max_blocks = size32(table.size(1));
    d.max_len_k = size32(table.size(1) * d.page_size);
    d.num_cache_tokens = kc.size(0);
    d.block_table = table.data_ptr<int32_t>();
    d.cu_seqlens_q = cu.data_ptr<int32_t>();
    d.seq_lens = lens.data_ptr<int32_t>();
    d.scale = 1.f;
    d.causal = 1;
    check(fn_append(&d, view(key), view(value), view(kc), view(vc), w.data, w.ld,
                    c10::cuda::getCurrentCUDAStream(key.device().index()).stream()),
          "hfan_paged_append");
    written(kc);
    written(vc);
    written(a[9]);
    Py_RETURN_NONE;
  });
}

// (q, key_cache, value_cache, block_table, cu_seqlens, lengths, page_size, max_q, max_k, normalizer, scale, causal,
//  key_weights) -> (o, stats)
PyObject* chunk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor q = rows(tensor(a[0]));
    const at::Tensor &kc = tensor(a[1]), &vc = tensor(a[2]);
    const c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor table = ints(tensor(a[3])), cu = ints(tensor(a[4])), lens = ints(tensor(a[5]));
    const Weights w(a[12]);
    hfan_chunk_desc d{};
    d.dtype = dtype_of(q);
    d.normalizer = int32(a[9]);
    d.batch = size32(table.size(0));
    d.heads_q = size32(q.size(1));
    d.heads_kv = size32(kc.size(1));
    d.head_dim = size32(q.size(2));
    d.total_q = size32(q.size(0));
    d.max_len_q = int32(a[7]);
    d.page_size = int32(a[6]);
    d.max_blocks = size32(table.size(1));
    d.max_len_k = int32(a[8]);
    d.num_cache_tokens = kc.size(0);
    d.block_table = table.data_ptr<int32_t>();
    d.cu_seqlens_q = cu.data_ptr<int32_t>();
    d.seq_lens = lens.data_ptr<int32_t>();
    const double scale = PyFloat_AsDouble(a[10]);
    if (scale == -1.0 && PyErr_Occurred()) throw PyFailure();
    d.scale = (float)scale;
    d.causal = PyObject_IsTrue(a[11]) == 1;
    const at::Tensor o = at::empty(q.sizes(), q.options());
    const at::Tensor stats = at::empty({2, q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
    const int64_t bytes = fn_bytes(&d, w.data != nullptr);
    at::Tensor ws;
    if (bytes > 0) ws = at::empty({bytes}, q.options().dtype(at::kByte));
    check(fn_chunk(&d, view(q), view(kc), view(vc), view(o), stats.data_ptr<float>(), w.data, w.ld,
                   bytes > 0 ? ws.data_ptr() : nullptr, bytes > 0 ? bytes : 0,
                   c10::cuda::getCurrentCUDAStream(q.device().index()).stream()),
          "hfan_paged_chunk_fwd");
    written(a[12]);
    return Py_BuildValue("NN", THPVariable_Wrap(o), THPVariable_Wrap(stats));
  });
}

// (key_cache, value_cache, key_weights, block_table, lengths, page_size, max_k, budget, recent) -> (lengths, kept)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const at::Tensor &kc = tensor(a[0]), &vc = tensor(a[1]);
    const c10::cuda::CUDAGuard guard(kc.device());
    const at::Tensor table = ints(tensor(a[3])), lens = ints(tensor(a[4]));
    const Weights w(a[2]);
    const int32_t budget = int32(a[7]);
    hfan_chunk_desc d{};
    d.dtype = dtype_of(kc);
    d.normalizer = HFAN_SOFTMAX1;
    d.batch = size32(table.size(0));
    d.heads_q = d.heads_kv = size32(kc.size(1));
    d.head_dim = size32(kc.size(2));
    d.page_size = int32(a[5]);
    d.max_blocks = size32(table.size(1));
    d.max_len_k = int32(a[6]);
    d.num_cache_tokens = kc.size(0);
    d.block_table = table.data_ptr<int32_t>();
    d.seq_lens = lens.data_ptr<int32_t>();
    d.scale = 1.f;
    d.causal = 1;
    const at::Tensor kept = at::empty({table.size(0), kc.size(1), budget}, table.options());
    const at::Tensor cut = at::empty({table.size(0)}, table.options());
    check(fn_evict(&d, view(kc), view(vc), w.data, w.ld, budget, int32(a[8]), kept.data_ptr<int32_t>(),
                   cut.data_ptr<int32_t>(), c10::cuda::getCurrentCUDAStream(kc.device().index()).stream()),
          "hfan_paged_evict");
    written(kc);
    written(vc);
    written(a[2]);
    return Py_BuildValue("NN", THPVariable_Wrap(cut), THPVariable_Wrap(kept));
  });
}

// Addresses of the five entry points, in the order of the declarations above.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    fn_append = reinterpret_cast<decltype(fn_append)>(integer(a[0]));
    fn_bytes = reinterpret_cast<decltype(fn_bytes)>(integer(a[1]));
    fn_chunk = reinterpret_cast<decltype(fn_chunk)>(integer(a[2]));
    fn_evict = reinterpret_cast<decltype(fn_evict)>(integer(a[3]));
    fn_error = reinterpret_cast<decltype(fn_error)>(integer(a[4]));
    Py_RETURN_NONE;
  });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(append), METHOD(chunk), METHOD(evict), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hfan_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hfan_torch(void) { return PyModule_Create(&module); }
