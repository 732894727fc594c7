// The calls of the cache in 8 bits (ops.py) for plain arguments: their checks and allocations in C++ instead of some eighty Python operations, which took 10 of a small
// call's 14 us.  A function here returns None where anything is out of the ordinary - another type, shape or layout than the call documents, another device than
// the current one, a refusal by the library - and then the caller goes through the checks in Python, which say what it is.  The library's entry points come as addresses.
// Pointers are taken while the interpreter's lock is held: tensors without storage (torch.vmap's, torch.func's) throw where theirs is asked for.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/b200_kv.h"

namespace {

decltype(&b200_rope_kv_append_q8) append_fn;
decltype(&b200_kv_gather_dense_q8) gather_fn;
decltype(&b200_paged_decode_attn_q8) decode_fn;
decltype(&b200_paged_decode_attn_q8_workspace) decode_ws_fn;
decltype(&b200_paged_prompt_attn_q8) prompt_fn;
decltype(&b200_paged_prompt_attn_q8_workspace) prompt_ws_fn;

int id_of(at::ScalarType t) {
  return t == at::kHalf ? B200_DTYPE_F16 : t == at::kFloat ? B200_DTYPE_F32 : t == at::kBFloat16 ? B200_DTYPE_BF16 : -1;
}
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }
bool whole_number(PyObject* o, int* to) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || v < 0 || v > INT32_MAX) return false;
  *to = static_cast<int>(v);
  return true;
}

struct Plain {
  int dev = -1;
  int64_t blocks = 0;
  int heads = 0, bs = 0, D = 0, codes = 0, B = 0, cols = 0, stride = 0;
  const at::Tensor *k_pool = nullptr, *v_pool = nullptr, *k_scale = nullptr, *v_scale = nullptr, *tables = nullptr;

  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided; }
  // pools, scales, tables
  bool cache(PyObject* const* a) {
    k_pool = tensor(a[0]), v_pool = tensor(a[1]), k_scale = tensor(a[2]), v_scale = tensor(a[3]), tables = tensor(a[4]);
    if (!k_pool || !v_pool || !k_scale || !v_scale || !tables) return false;
    if (!k_pool->is_cuda() || k_pool->get_device() != c10::cuda::current_device()) return false;
    dev = k_pool->get_device();
    if (!here(*k_pool) || !here(*v_pool) || !here(*k_scale) || !here(*v_scale) || !here(*tables)) return false;
    const at::ScalarType kind = k_pool->scalar_type();
    codes = kind == at::kChar ? B200_CODES_INT8 : kind == at::kFloat8_e4m3fn ? B200_CODES_E4M3 : 0;
    if (!codes || v_pool->scalar_type() != kind || k_pool->dim() != 4 || !k_pool->is_contiguous() || !v_pool->is_contiguous() || v_pool->sizes() != k_pool->sizes()) return false;
    blocks = k_pool->size(0);
    if (k_pool->size(1) > INT32_MAX || k_pool->size(2) > INT32_MAX || k_pool->size(3) > INT32_MAX) return false;
    heads = static_cast<int>(k_pool->size(1)), bs = static_cast<int>(k_pool->size(2)), D = static_cast<int>(k_pool->size(3));
    for (const at::Tensor* s : {k_scale, v_scale})
      if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != blocks || s->size(1) != heads || !s->is_contiguous()) return false;
    if (tables->scalar_type() != at::kInt || tables->dim() != 2 || tables->size(1) < 1 || tables->size(0) > INT32_MAX || tables->size(1) > INT32_MAX) return false;
    B = static_cast<int>(tables->size(0)), cols = static_cast<int>(tables->size(1));
    if (cols > 1 && tables->stride(1) != 1) return false;
    const int64_t apart = B > 1 ? tables->stride(0) : cols;
    if (apart < 0 || apart > INT32_MAX) return false;
    stride = static_cast<int>(apart);
    return true;
  }
  bool whole(const at::Tensor* t, int64_t n) const {       // a contiguous vector of whole numbers
    return t && here(*t) && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
  }
  // [n, heads, D], the heads contiguous inside a row
  bool rows(const at::Tensor* t, int64_t n, at::ScalarType kind, int64_t* apart) const {
    if (!t || !here(*t) || t->scalar_type() != kind || t->dim() != 3 || t->size(0) != n || t->size(2) != D) return false;
    if (n > 0 && (t->stride(2) != 1 || t->stride(1) != D)) return false;
    *apart = n > 1 ? t->stride(0) : t->size(1) * D;
    return *apart >= 0;
  }
  // of pools, scales and tables; may throw
  void *kp = nullptr, *vp = nullptr;
  float *ks = nullptr, *vs = nullptr;
  const int32_t* rows_of_tables = nullptr;
  void pointers() {
    kp = k_pool->data_ptr(), vp = v_pool->data_ptr(), ks = static_cast<float*>(k_scale->data_ptr()), vs = static_cast<float*>(v_scale->data_ptr());
    rows_of_tables = whole_numbers(tables);
  }
  static const int32_t* whole_numbers(const at::Tensor* t) { return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; }
  at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType kind) const { return at::empty(sizes, k_pool->options().dtype(kind)); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }
};

// q, k, v, cos, sin (q, cos and sin or none of them), pools, scales, tables, lens, row_starts or None, max_new or None -> rotated queries
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plain c;
  if (count != 13 || !c.cache(a + 5)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *cos = tensor(a[3]), *sin = tensor(a[4]), *lens = tensor(a[10]), *starts = tensor(a[11]);
  if (!q || !k || !v || !cos || !sin || !lens || (!starts && a[11] != Py_None) || k->dim() != 3) Py_RETURN_NONE;
  const int64_t n = k->size(0);
  const at::ScalarType kind = k->scalar_type();
  const int dtype = id_of(kind);
  int64_t qs, ks, vs;
  if (dtype < 0 || n > INT32_MAX || !c.rows(q, n, kind, &qs) || !c.rows(k, n, kind, &ks) || !c.rows(v, n, kind, &vs) || k->size(1) != c.heads || v->size(1) != c.heads ||
      q->size(1) > INT32_MAX)
    Py_RETURN_NONE;
  for (const at::Tensor* t : {cos, sin})
    if (!c.here(*t) || t->scalar_type() != kind || t->dim() != 2 || t->size(0) != n || t->size(1) != c.D || !t->is_contiguous()) Py_RETURN_NONE;
  if (!c.whole(lens, c.B) || (starts ? !c.whole(starts, c.B + 1ll) : n != c.B)) Py_RETURN_NONE;
  int most = static_cast<int>(n);
  if (a[12] != Py_None && !whole_number(a[12], &most)) Py_RETURN_NONE;
  at::Tensor out = c.fresh(q->sizes(), kind);
  c.pointers();
  void *op = out.data_ptr(), *stream = c.stream();
  const void *qp = q->data_ptr(), *kp = k->data_ptr(), *vp = v->data_ptr(), *cp = cos->data_ptr(), *sp = sin->data_ptr();
  const int32_t *contexts = c.whole_numbers(lens), *firsts = c.whole_numbers(starts);
  const int Hq = static_cast<int>(q->size(1));
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = append_fn(op, static_cast<int64_t>(Hq) * c.D, qp, qs, kp, ks, vp, vs, cp, sp, c.kp, c.vp, c.ks, c.vs, c.rows_of_tables, c.stride, c.cols, contexts, firsts, c.B, static_cast<int>(n), most, Hq,
                 c.heads, c.D, c.bs, c.blocks, c.codes, dtype, stream);
  Py_END_ALLOW_THREADS;
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// pools, scales, tables, n_tokens, the library's number of the dtype -> (k, v)
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  Plain c;
  int n, dtype;
  if (count != 7 || !c.cache(a) || !whole_number(a[5], &n) || !whole_number(a[6], &dtype) || n > static_cast<int64_t>(c.cols) * c.bs) Py_RETURN_NONE;
  const at::ScalarType kind = dtype == B200_DTYPE_F16 ? at::kHalf : dtype == B200_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
  at::Tensor k = c.fresh({c.B, c.heads, n, c.D}, kind), v = c.fresh({c.B, c.heads, n, c.D}, kind);
  c.pointers();
  void *k_out = k.data_ptr(), *v_out = v.data_ptr(), *stream = c.stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = gather_fn(k_out, v_out, c.kp, c.vp, c.ks, c.vs, c.rows_of_tables, c.stride, c.cols, c.B, n, c.heads, c.D, c.bs, c.blocks, c.codes, dtype, stream);
  Py_END_ALLOW_THREADS;
  if (rc != 0) Py_RETURN_NONE;
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(v)));
  return pair;
  END_HANDLE_TH_ERRORS
}

// q, pools, scales, tables, lens, [row_starts, max_new,] max_context_len, scale -> out
PyObject* attention(PyObject* const* a, Py_ssize_t count, bool several) {
  Plain c;
  if (count != (several ? 11 : 9) || !c.cache(a + 1)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *lens = tensor(a[6]), *starts = several ? tensor(a[7]) : nullptr;
  int most = 1, longest;
  if (!q || q->dim() != 3 || !whole_number(a[several ? 9 : 7], &longest) || (several && (!starts || !whole_number(a[8], &most)))) Py_RETURN_NONE;
  PyObject* by = a[several ? 10 : 8];
  if (by != Py_None && !PyFloat_CheckExact(by)) Py_RETURN_NONE;
  const int64_t n = q->size(0), heads = q->size(1);
  const int dtype = id_of(q->scalar_type());
  int64_t qs;
  if (dtype < 0 || n > INT32_MAX || heads > INT32_MAX || heads == 0 || c.heads == 0 || heads % c.heads || !c.rows(q, n, q->scalar_type(), &qs) || !c.whole(lens, c.B) ||
      (several ? !c.whole(starts, c.B + 1ll) : n != c.B))
    Py_RETURN_NONE;
  const float scale = by == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(c.D))) : static_cast<float>(PyFloat_AS_DOUBLE(by));
  const int Hq = static_cast<int>(heads);
  at::Tensor out = c.fresh(q->sizes(), q->scalar_type()), workspace;
  const size_t need = several ? prompt_ws_fn(c.B, most, Hq, c.heads, c.D, c.bs, longest, dtype) : decode_ws_fn(c.B, Hq, c.heads, c.D, c.bs, longest, dtype);
  if (need) workspace = c.fresh({static_cast<int64_t>(need)}, at::kByte);
  c.pointers();
  void *op = out.data_ptr(), *stream = c.stream(), *ws = need ? workspace.data_ptr() : nullptr;
  const void* qp = q->data_ptr();
  const int32_t *contexts = c.whole_numbers(lens), *firsts = c.whole_numbers(starts);
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = several ? prompt_fn(op, qp, qs, c.kp, c.vp, c.ks, c.vs, c.rows_of_tables, c.stride, c.cols, contexts, firsts, c.B, static_cast<int>(n), most, Hq, c.heads, c.D, c.bs, c.blocks, scale, longest,
                           ws, need, c.codes, dtype, 0u, stream)
               : decode_fn(op, qp, qs, c.kp, c.vp, c.ks, c.vs, c.rows_of_tables, c.stride, c.cols, contexts, c.B, Hq, c.heads, c.D, c.bs, c.blocks, scale, longest, ws, need, c.codes, dtype, 0u, stream);
  Py_END_ALLOW_THREADS;
  if (rc != 0) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
}
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  return attention(a, count, false);
  END_HANDLE_TH_ERRORS
}
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  return attention(a, count, true);
  END_HANDLE_TH_ERRORS
}

// the library's entry points, in the order of their names above
PyObject* entry_points(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 6) {
    PyErr_SetString(PyExc_TypeError, "six addresses");
    return nullptr;
  }
  void* at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  append_fn = reinterpret_cast<decltype(append_fn)>(at[0]);
  gather_fn = reinterpret_cast<decltype(gather_fn)>(at[1]);
  decode_fn = reinterpret_cast<decltype(decode_fn)>(at[2]);
  decode_ws_fn = reinterpret_cast<decltype(decode_ws_fn)>(at[3]);
  prompt_fn = reinterpret_cast<decltype(prompt_fn)>(at[4]);
  prompt_ws_fn = reinterpret_cast<decltype(prompt_ws_fn)>(at[5]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"append", FAST(append)}, {"gather", FAST(gather)}, {"decode", FAST(decode)}, {"prompt", FAST(prompt)}, {"entry_points", FAST(entry_points)}, {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fast_calls() { return PyModule_Create(&module); }
