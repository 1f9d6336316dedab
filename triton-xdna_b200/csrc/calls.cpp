// The host side of a paged or beam step's calls, for Python.  A step of single tokens is
// bound by the host: of the 18 us between two calls of paged_attention from Python
// the GPU worked 8, the two launches took 6, and looking at ten tensors through
// the interpreter (shape, strides, type, address: some 50 attribute reads) with
// ctypes' conversions the rest.  Here a call costs little more than its launches: with
// the same kernels 8.6 us (write and reading back 23.8 -> 8.4, select 21.4 -> 9.5).
//
// Each function takes a call if everything about it is as xb200/ops.py asks, makes
// it through the same C entry point and says so; anything else (another type, a
// wrong shape, tensors of another device than the current one, arguments that the
// library refuses) it leaves alone, before anything is launched, to the function of
// the same name there, which has the checks one by one and their messages.  An
// error of CUDA's, which may come after a launch, is raised here: the call is not
// made again.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "xb200.h"

namespace {

// Entry points of the library that xb200/_lib.py has loaded (null before that: every call is left alone).
struct Entries {
  decltype(&xb_paged_attention_workspace_size) attention_size;
  decltype(&xb_paged_attention_bf16) attention;
  decltype(&xb_paged_attention_q8_workspace_size) attention8_size;
  decltype(&xb_paged_attention_q8) attention8;
  decltype(&xb_paged_rope_kv_bf16) rope_kv;
  decltype(&xb_paged_rope_kv_q8) rope_kv8;
  decltype(&xb_paged_read_kv) read_kv;
  decltype(&xb_beam_select_workspace_size) beam_size;
  decltype(&xb_beam_select) beam;
} entry = {};
PyObject* error_type = nullptr;  // xb200/_lib.py's XbError
bool bound = false;

PyObject* bind(PyObject*, PyObject* addresses) {
  auto get = [&](auto& fn, const char* name) {
    PyObject* v = PyDict_GetItemString(addresses, name);
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "no address of %s", name);
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    return p != nullptr;
  };
  if (!PyDict_Check(addresses)) {
    PyErr_SetString(PyExc_TypeError, "bind takes a dict");
    return nullptr;
  }
  PyObject* type = PyDict_GetItemString(addresses, "error");
  if (!type || !PyExceptionClass_Check(type)) {
    PyErr_SetString(PyExc_RuntimeError, "no type of errors");
    return nullptr;
  }
  Py_INCREF(type);
  Py_XSETREF(error_type, type);
  bound = get(entry.attention_size, "xb_paged_attention_workspace_size") &&
          get(entry.attention, "xb_paged_attention_bf16") &&
          get(entry.attention8_size, "xb_paged_attention_q8_workspace_size") &&
          get(entry.attention8, "xb_paged_attention_q8") && get(entry.rope_kv, "xb_paged_rope_kv_bf16") &&
          get(entry.rope_kv8, "xb_paged_rope_kv_q8") && get(entry.read_kv, "xb_paged_read_kv") &&
          get(entry.beam_size, "xb_beam_select_workspace_size") && get(entry.beam, "xb_beam_select");
  if (!bound) return nullptr;
  Py_RETURN_NONE;
}

// Arguments as tensors of one device.  `ok` turns false at the first that is not one.
struct Args {
  PyObject* const* a;
  int device = -1;
  bool ok = true;

  const at::Tensor& operator()(int i) {
    static const at::Tensor nothing;
    if (!THPVariable_CheckExact(a[i])) {
      ok = false;
      return nothing;
    }
    const at::Tensor& t = THPVariable_Unpack(a[i]);
    if (!t.is_cuda() || t.layout() != at::kStrided || (device >= 0 && t.get_device() != device)) {
      ok = false;
      return nothing;
    }
    device = t.get_device();
    return t;
  }
  const at::Tensor* optional(int i) { return a[i] == Py_None ? nullptr : &(*this)(i); }
  bool here() const { return ok && device == c10::cuda::current_device(); }
};

// xb200/ops.py's _page_args.  kv8.dtype: XB_DT_BF16 for pages without exponents.
bool page_args(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& q_start,
               const at::Tensor& kv_len, const at::Tensor* ks, const at::Tensor* vs, xb_paged_kv8& kv8) {
  const at::ScalarType type = k.scalar_type();
  const bool coded = type == at::kChar || type == at::kFloat8_e4m3fn;
  if ((!coded && type != at::kBFloat16) || v.scalar_type() != type || coded != (ks != nullptr) ||
      coded != (vs != nullptr) || table.scalar_type() != at::kInt || q_start.scalar_type() != at::kInt ||
      kv_len.scalar_type() != at::kInt)
    return false;
  if (k.dim() != 4 || v.sizes() != k.sizes() || kv_len.dim() != 1 || table.dim() != 2 || q_start.dim() != 1)
    return false;
  const int64_t n = k.size(0), h = k.size(1), p = k.size(2), d = k.size(3), B = table.size(0), cols = table.size(1);
  if (kv_len.size(0) != B || q_start.size(0) != B + 1 || cols == 0 || (table.stride(1) != 1 && cols > 1) ||
      !q_start.is_contiguous() || !kv_len.is_contiguous() || ((k.stride(3) != 1 || v.stride(3) != 1) && d > 1))
    return false;
  const int64_t any = h * p * d;  // the stride of a dimension of one is arbitrary
  kv8 = xb_paged_kv8{};
  xb_paged_kv& kv = kv8.kv;
  kv.k_pages = k.data_ptr();
  kv.v_pages = v.data_ptr();
  kv.page_table = static_cast<const int32_t*>(table.data_ptr());
  kv.q_start = static_cast<const int32_t*>(q_start.data_ptr());
  kv.kv_len = static_cast<const int32_t*>(kv_len.data_ptr());
  kv.n_pages = n;
  kv.n_kv_head = h;
  kv.page_size = p;
  kv.head_dim = d;
  kv.batch = B;
  kv.max_pages = cols;
  kv.ld_table = B > 1 ? table.stride(0) : cols;
  kv.k_page = n == 1 ? any : k.stride(0);
  kv.k_head = h == 1 ? any : k.stride(1);
  kv.k_row = p == 1 ? any : k.stride(2);
  kv.v_page = n == 1 ? any : v.stride(0);
  kv.v_head = h == 1 ? any : v.stride(1);
  kv.v_row = p == 1 ? any : v.stride(2);
  kv8.dtype = XB_DT_BF16;
  if (!coded) return true;
  kv8.dtype = type == at::kChar ? XB_DT_I8 : XB_DT_F8E4M3;
  for (const at::Tensor* t : {ks, vs})
    if (t->scalar_type() != at::kByte || t->sizes() != k.sizes().slice(0, 3) || (t->stride(2) != 1 && p > 1))
      return false;
  kv8.k_scale = static_cast<uint8_t*>(ks->data_ptr());
  kv8.v_scale = static_cast<uint8_t*>(vs->data_ptr());
  kv8.ks_page = n == 1 ? h * p : ks->stride(0);
  kv8.ks_head = h == 1 ? p : ks->stride(1);
  kv8.vs_page = n == 1 ? h * p : vs->stride(0);
  kv8.vs_head = h == 1 ? p : vs->stride(1);
  return true;
}

// xb200/ops.py's _token_rows: the pitch of `tokens` rows of `row` bf16 elements, -1 for anything else.
int64_t token_rows(const at::Tensor& t, int64_t tokens, int64_t row) {
  if (t.scalar_type() != at::kBFloat16) return -1;
  const int64_t dims = t.dim();
  if ((dims != 2 && dims != 3) || t.size(0) != tokens || (dims == 2 ? t.size(1) : t.size(1) * t.size(2)) != row)
    return -1;
  if (tokens && (t.stride(-1) != 1 || (dims == 3 && t.size(1) > 1 && t.stride(1) != t.size(2)))) return -1;
  return tokens > 1 ? t.stride(0) : row;
}

// xb200/ops.py's _apart: one of two [tokens, row] bf16 tensors ends before the other starts, or they are other columns
// of the same rows.
bool apart(const void* p, int64_t ld_p, int64_t row_p, const void* q, int64_t ld_q, int64_t row_q, int64_t tokens) {
  const auto x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
  if (tokens == 0 || x + 2 * ((tokens - 1) * ld_p + row_p) <= y || y + 2 * ((tokens - 1) * ld_q + row_q) <= x)
    return true;
  if (ld_p != ld_q || ld_p <= 0) return false;
  int64_t off = (int64_t)(y - x) / 2 % ld_p;  // both are multiples of two
  if (off < 0) off += ld_p;
  return off >= row_p && off + row_q <= ld_p;
}

struct Error {
  char text[256] = "";
};

// Whether an entry point's answer is that it made the call; false: it refused its arguments, and has launched nothing.
// Anything else raises XbError.
bool made(const char* name, int rc, const Error& err) {
  if (rc == XB_OK) return true;
  if (rc == XB_ERR_INVALID || rc == XB_ERR_UNSUPPORTED) return false;
  if (PyObject* e = PyObject_CallFunction(error_type, "sis", name, rc, err.text)) {
    PyErr_SetObject(error_type, e);
    Py_DECREF(e);
  }
  throw python_error();
}

// paged_attention(q, k_pages, v_pages, out, page_table, q_start, kv_len, scale, k_scale, v_scale): whether it was done
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (!bound || count != 10 || !PyFloat_CheckExact(a[7])) Py_RETURN_FALSE;
  Args arg{a};
  const at::Tensor &q = arg(0), &k = arg(1), &v = arg(2), &out = arg(3), &table = arg(4), &q_start = arg(5),
                   &kv_len = arg(6);
  const at::Tensor *ks = arg.optional(8), *vs = arg.optional(9);
  xb_paged_kv8 kv;
  if (!arg.here() || !page_args(k, v, table, q_start, kv_len, ks, vs, kv)) Py_RETURN_FALSE;
  if (q.dim() != 3 || q.size(2) != kv.kv.head_dim) Py_RETURN_FALSE;
  const int64_t T = q.size(0), H = q.size(1), row = H * kv.kv.head_dim;
  const int64_t ld_q = token_rows(q, T, row), ld_out = token_rows(out, T, row);
  if (ld_q < 0 || ld_out < 0) Py_RETURN_FALSE;
  const void* pq = q.data_ptr();
  void* po = out.data_ptr();
  if (!apart(pq, ld_q, row, po, ld_out, row, T)) Py_RETURN_FALSE;
  const bool coded = kv.dtype != XB_DT_BF16;
  Error err;
  size_t need = 0;
  int rc = coded ? entry.attention8_size(T, kv.kv.batch, H, kv.kv.n_kv_head, kv.kv.n_pages, kv.kv.page_size,
                                         kv.kv.max_pages, &need, err.text, sizeof(err.text))
                 : entry.attention_size(T, kv.kv.batch, H, kv.kv.n_kv_head, &need, err.text, sizeof(err.text));
  if (!made(coded ? "xb_paged_attention_q8_workspace_size" : "xb_paged_attention_workspace_size", rc, err))
    Py_RETURN_FALSE;
  const float scale = (float)PyFloat_AS_DOUBLE(a[7]);
  // of this call alone: the caching allocator orders its reuse on the stream, and a captured graph keeps its own
  c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(need);
  void* stream = c10::cuda::getCurrentCUDAStream(arg.device).stream();
  Py_BEGIN_ALLOW_THREADS
  rc = coded ? entry.attention8(pq, po, &kv, T, H, ld_q, ld_out, scale, ws.get(), need, stream, err.text,
                                sizeof(err.text))
             : entry.attention(pq, po, &kv.kv, T, H, ld_q, ld_out, scale, ws.get(), need, stream, err.text,
                               sizeof(err.text));
  Py_END_ALLOW_THREADS
  return PyBool_FromLong(made(coded ? "xb_paged_attention_q8" : "xb_paged_attention_bf16", rc, err));
  END_HANDLE_TH_ERRORS
}

// paged_rope_kv(qkv, cos_t, sin_t, q_out, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale): the same
PyObject* paged_rope_kv(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (!bound || count != 11 || (a[1] == Py_None) != (a[2] == Py_None)) Py_RETURN_FALSE;
  Args arg{a};
  const at::Tensor &qkv = arg(0), &q = arg(3), &k = arg(4), &v = arg(5), &table = arg(6), &q_start = arg(7),
                   &kv_len = arg(8);
  const at::Tensor *cos_t = arg.optional(1), *sin_t = arg.optional(2), *ks = arg.optional(9), *vs = arg.optional(10);
  xb_paged_kv8 kv;
  if (!arg.here() || !page_args(k, v, table, q_start, kv_len, ks, vs, kv)) Py_RETURN_FALSE;
  const int64_t D = kv.kv.head_dim;
  if (q.dim() != 3 || q.size(2) != D) Py_RETURN_FALSE;
  int64_t rows = 0;
  if (cos_t) {
    for (const at::Tensor* t : {cos_t, sin_t})
      if (t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) != D || !t->is_contiguous()) Py_RETURN_FALSE;
    if (cos_t->sizes() != sin_t->sizes()) Py_RETURN_FALSE;
    rows = cos_t->size(0);
    if (rows == 0) Py_RETURN_FALSE;
  }
  const int64_t T = q.size(0), H = q.size(1), row = (H + 2 * kv.kv.n_kv_head) * D;
  const int64_t ld_qkv = token_rows(qkv, T, row), ld_q = token_rows(q, T, H * D);
  if (ld_qkv < 0 || ld_q < 0) Py_RETURN_FALSE;
  const void* px = qkv.data_ptr();
  void* pq = q.data_ptr();
  if (!apart(px, ld_qkv, row, pq, ld_q, H * D, T)) Py_RETURN_FALSE;
  const float* c = cos_t ? static_cast<const float*>(cos_t->data_ptr()) : nullptr;
  const float* s = sin_t ? static_cast<const float*>(sin_t->data_ptr()) : nullptr;
  void* stream = c10::cuda::getCurrentCUDAStream(arg.device).stream();
  Error err;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = kv.dtype != XB_DT_BF16
           ? entry.rope_kv8(px, c, s, pq, &kv, T, H, rows, ld_qkv, ld_q, stream, err.text, sizeof(err.text))
           : entry.rope_kv(px, c, s, pq, &kv.kv, T, H, rows, ld_qkv, ld_q, stream, err.text, sizeof(err.text));
  Py_END_ALLOW_THREADS
  return PyBool_FromLong(made(kv.dtype != XB_DT_BF16 ? "xb_paged_rope_kv_q8" : "xb_paged_rope_kv_bf16", rc, err));
  END_HANDLE_TH_ERRORS
}

// paged_read_kv(k_out, v_out, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale): the same
PyObject* paged_read_kv(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (!bound || count != 9) Py_RETURN_FALSE;
  Args arg{a};
  const at::Tensor &k_out = arg(0), &v_out = arg(1), &k = arg(2), &v = arg(3), &table = arg(4), &q_start = arg(5),
                   &kv_len = arg(6);
  const at::Tensor *ks = arg.optional(7), *vs = arg.optional(8);
  xb_paged_kv8 kv;
  if (!arg.here() || !page_args(k, v, table, q_start, kv_len, ks, vs, kv) || k_out.dim() == 0) Py_RETURN_FALSE;
  const int64_t T = k_out.size(0), row = kv.kv.n_kv_head * kv.kv.head_dim;
  const int64_t ld_k = token_rows(k_out, T, row), ld_v = token_rows(v_out, T, row);
  if (ld_k < 0 || ld_v < 0) Py_RETURN_FALSE;
  void *pk = k_out.data_ptr(), *pv = v_out.data_ptr();
  if (!apart(pk, ld_k, row, pv, ld_v, row, T)) Py_RETURN_FALSE;
  void* stream = c10::cuda::getCurrentCUDAStream(arg.device).stream();
  Error err;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = entry.read_kv(pk, pv, &kv, T, ld_k, ld_v, stream, err.text, sizeof(err.text));
  Py_END_ALLOW_THREADS
  return PyBool_FromLong(made("xb_paged_read_kv", rc, err));
  END_HANDLE_TH_ERRORS
}

// beam_select(logits, scores, count): (values, parents, tokens), or None if it was not done
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t given) {
  HANDLE_TH_ERRORS
  if (!bound || given != 3 || !PyLong_CheckExact(a[2])) Py_RETURN_NONE;
  const int64_t count = PyLong_AsLongLong(a[2]);
  if (count <= 0) {  // also what does not fit
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  Args arg{a};
  const at::Tensor &logits = arg(0), &scores = arg(1);
  if (!arg.here()) Py_RETURN_NONE;
  const at::ScalarType type = logits.scalar_type();
  if ((type != at::kFloat && type != at::kBFloat16) || scores.scalar_type() != at::kFloat || logits.dim() != 2 ||
      scores.dim() != 2 || logits.size(0) != scores.numel())
    Py_RETURN_NONE;
  const int64_t G = scores.size(0), K = scores.size(1), V = logits.size(1);
  if ((logits.stride(1) != 1 && V > 1) || (scores.stride(1) != 1 && K > 1)) Py_RETURN_NONE;
  Error err;
  size_t need = 0;
  int rc = entry.beam_size(G, K, V, count, &need, err.text, sizeof(err.text));
  if (!made("xb_beam_select_workspace_size", rc, err)) Py_RETURN_NONE;
  const at::TensorOptions on = at::TensorOptions().device(logits.device());
  at::Tensor values = at::empty({G, count}, on.dtype(at::kFloat));
  at::Tensor parents = at::empty({G, count}, on.dtype(at::kLong)), tokens = at::empty({G, count}, on.dtype(at::kLong));
  c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(need);  // as in paged_attention
  const void* x = logits.data_ptr();
  const float* s = static_cast<const float*>(scores.data_ptr());
  float* to_values = static_cast<float*>(values.data_ptr());
  int64_t* to_parents = static_cast<int64_t*>(parents.data_ptr());
  int64_t* to_tokens = static_cast<int64_t*>(tokens.data_ptr());
  const int64_t ld = G * K > 1 ? logits.stride(0) : V, ld_scores = G > 1 ? scores.stride(0) : K;
  void* stream = c10::cuda::getCurrentCUDAStream(arg.device).stream();
  Py_BEGIN_ALLOW_THREADS
  rc = entry.beam(x, s, G, K, V, ld, ld_scores, count, type == at::kFloat ? XB_DT_F32 : XB_DT_BF16, to_values,
                  to_parents, to_tokens, ws.get(), need, stream, err.text, sizeof(err.text));
  Py_END_ALLOW_THREADS
  if (!made("xb_beam_select", rc, err)) Py_RETURN_NONE;
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  at::Tensor* results[3] = {&values, &parents, &tokens};
  for (int i = 0; i < 3; ++i) {
    PyObject* t = THPVariable_Wrap(std::move(*results[i]));
    if (!t) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i, t);
  }
  return out;
  END_HANDLE_TH_ERRORS
}

PyCFunction function(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "Addresses of the library's entry points, and the type of its errors (error)."},
    {"paged_attention", function(paged_attention), METH_FASTCALL, "Whether it made the call."},
    {"paged_rope_kv", function(paged_rope_kv), METH_FASTCALL, "Whether it made the call."},
    {"paged_read_kv", function(paged_read_kv), METH_FASTCALL, "Whether it made the call."},
    {"beam_select", function(beam_select), METH_FASTCALL, "What it selected, None if it did not make the call."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", "Calls of operators without the interpreter.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", XB_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
