// dtt._tensorlist: what a multi-tensor call has to know of its lists of tensors -- addresses, element counts, types, device,
// memory order -- read in one pass over each list.  From Python this costs about 4 us per parameter of an AdamW step (five
// tensors with seven questions each): 1.1 ms for 301 small tensors, whose kernels take 56 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/core/Tensor.h>
#include <algorithm>
#include <exception>
#include <utility>

namespace {

enum { kOther = -1, kF32 = 0, kBf16 = 1, kF16 = 2, kU8 = 3, kI16 = 4 };
enum { kNone = -3, kSeveral = -2, kHost = -1 };   // devices beside an index

int type_code(const at::Tensor& t) {
  if (t.layout() != at::kStrided || t.is_neg()) return kOther;   // (a negated view's memory is not its values)
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kBFloat16: return kBf16;
    case at::kHalf: return kF16;
    case at::kByte: return kU8;
    case at::kShort: return kI16;
    default: return kOther;
  }
}

// one run of memory, in whatever order of the dimensions
bool dense(const at::Tensor& t) {
  if (t.is_contiguous()) return true;
  const auto sizes = t.sizes(), strides = t.strides();
  if (sizes.size() > 16) return false;
  std::pair<int64_t, int64_t> d[16];
  int n = 0;
  for (size_t i = 0; i < sizes.size(); ++i)
    if (sizes[i] != 1) d[n++] = {strides[i], sizes[i]};
  std::sort(d, d + n);
  int64_t expected = 1;
  for (int i = 0; i < n; ++i) {
    if (d[i].first != expected) return false;
    expected *= d[i].second;
  }
  return true;
}

// the same element at the same place of memory, for equal shapes and a dense `a`
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  if (a.is_contiguous() && b.is_contiguous()) return true;
  const auto sizes = a.sizes(), x = a.strides(), y = b.strides();
  for (size_t i = 0; i < sizes.size(); ++i)
    if (sizes[i] != 1 && x[i] != y[i]) return false;
  return true;
}

bool is_list(PyObject* o, const char* what) {
  if (PyList_Check(o)) return true;
  PyErr_Format(PyExc_TypeError, "%s: expected a list (got %s)", what, Py_TYPE(o)->tp_name);
  return false;
}

// describe(list) -> (addresses, element counts, type codes: bytes of int64 / int64 / int32, device, common type or -2, first entry that
// is not dense or -1)
PyObject* describe(PyObject*, PyObject* list) {
  if (!is_list(list, "describe")) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  PyObject* ptrs = PyBytes_FromStringAndSize(nullptr, n * 8);
  PyObject* counts = PyBytes_FromStringAndSize(nullptr, n * 8);
  PyObject* types = PyBytes_FromStringAndSize(nullptr, n * 4);
  if (!ptrs || !counts || !types) {
    Py_XDECREF(ptrs); Py_XDECREF(counts); Py_XDECREF(types);
    return nullptr;
  }
  uint64_t* p = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(ptrs));
  int64_t* c = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(counts));
  int32_t* ty = reinterpret_cast<int32_t*>(PyBytes_AS_STRING(types));
  long device = kNone, type = -2, odd = -1;
  bool failed = false;
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(list, i);
      if (!THPVariable_Check(o)) {
        PyErr_Format(PyExc_TypeError, "expected tensors (got %s)", Py_TYPE(o)->tp_name);
        failed = true;
        break;
      }
      const at::Tensor& t = THPVariable_Unpack(o);
      const int code = type_code(t);
      const long d = t.is_cuda() ? (long)t.get_device() : kHost;
      ty[i] = code;
      type = i == 0 ? code : type == code ? type : -2;
      device = i == 0 || d == device ? d : d == kHost || device == kHost ? kHost : kSeveral;
      if (code == kOther) { p[i] = 0; c[i] = 0; continue; }
      p[i] = d == kHost ? 0 : reinterpret_cast<uint64_t>(t.data_ptr());
      c[i] = t.numel();
      if (odd < 0 && !dense(t)) odd = (long)i;
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    failed = true;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "describe: unknown C++ exception");
    failed = true;
  }
  if (failed) {
    Py_DECREF(ptrs); Py_DECREF(counts); Py_DECREF(types);
    return nullptr;
  }
  return Py_BuildValue("(NNNlll)", ptrs, counts, types, device, type, odd);
}

// differ(a, b) -> -1, or the first i where b[i] has not a[i]'s shape (2 i) or not its memory order (2 i + 1); lists of tensors of one
// length that describe() has seen
PyObject* differ(PyObject*, PyObject* args) {
  PyObject *a, *b;
  if (!PyArg_ParseTuple(args, "OO", &a, &b) || !is_list(a, "differ") || !is_list(b, "differ")) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(a);
  if (PyList_GET_SIZE(b) != n) {
    PyErr_SetString(PyExc_ValueError, "differ: lists of different lengths");
    return nullptr;
  }
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *oa = PyList_GET_ITEM(a, i), *ob = PyList_GET_ITEM(b, i);
      if (!THPVariable_Check(oa) || !THPVariable_Check(ob)) {
        PyErr_SetString(PyExc_TypeError, "expected tensors");
        return nullptr;
      }
      const at::Tensor &x = THPVariable_Unpack(oa), &y = THPVariable_Unpack(ob);
      if (x.sizes() != y.sizes()) return PyLong_FromSsize_t(2 * i);
      if (!same_order(x, y)) return PyLong_FromSsize_t(2 * i + 1);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "differ: unknown C++ exception");
    return nullptr;
  }
  return PyLong_FromLong(-1);
}

bool rows_for(const at::Tensor& t, const at::Tensor& rows, long block) {
  return type_code(rows) == kI16 && rows.dim() == 2 && rows.size(0) == (t.numel() + block - 1) / block && rows.size(1) == 2 && rows.is_contiguous();
}

// rows_of(a, b, block) -> -1, or the first i where b[i] is not a contiguous int16 matrix of two columns and a row for every `block`
// elements of a[i]
PyObject* rows_of(PyObject*, PyObject* args) {
  PyObject *a, *b;
  long block;
  if (!PyArg_ParseTuple(args, "OOl", &a, &b, &block) || !is_list(a, "rows_of") || !is_list(b, "rows_of")) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(a);
  if (PyList_GET_SIZE(b) != n || block < 1) {
    PyErr_SetString(PyExc_ValueError, "rows_of: lists of different lengths");
    return nullptr;
  }
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject *oa = PyList_GET_ITEM(a, i), *ob = PyList_GET_ITEM(b, i);
      if (!THPVariable_Check(oa) || !THPVariable_Check(ob)) {
        PyErr_SetString(PyExc_TypeError, "expected tensors");
        return nullptr;
      }
      if (!rows_for(THPVariable_Unpack(oa), THPVariable_Unpack(ob), block)) return PyLong_FromSsize_t(i);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "rows_of: unknown C++ exception");
    return nullptr;
  }
  return PyLong_FromLong(-1);
}

// step_lists([params, grads, steps, m, v] or [..., bases], type code of the moments, block) -> None, or (type code, device, tuple of
// address arrays, element counts): what a step hands to the library where everything is as it has to be -- one type among the parameters,
// dense, gradients and moments in their shape and order, one device.  None says only that it is not; the caller looks closer.
PyObject* step_lists(PyObject*, PyObject* args) {
  PyObject* lists;
  long moment, block;
  if (!PyArg_ParseTuple(args, "Oll", &lists, &moment, &block) || !is_list(lists, "step_lists")) return nullptr;
  const Py_ssize_t k = PyList_GET_SIZE(lists);
  PyObject* l[6];
  if (k != 5 && k != 6) {
    PyErr_SetString(PyExc_ValueError, "step_lists: five or six lists");
    return nullptr;
  }
  for (Py_ssize_t j = 0; j < k; ++j) {
    l[j] = PyList_GET_ITEM(lists, j);
    if (!is_list(l[j], "step_lists")) return nullptr;
    if (PyList_GET_SIZE(l[j]) != PyList_GET_SIZE(l[0])) Py_RETURN_NONE;
  }
  const Py_ssize_t n = PyList_GET_SIZE(l[0]);
  if (n == 0) Py_RETURN_NONE;
  PyObject* out = PyTuple_New(k);
  PyObject* counts = PyBytes_FromStringAndSize(nullptr, n * 8);
  uint64_t* at[6];
  bool whole = out && counts;
  for (Py_ssize_t j = 0; whole && j < k; ++j) {
    PyObject* b = PyBytes_FromStringAndSize(nullptr, n * 8);
    if (b) {
      PyTuple_SET_ITEM(out, j, b);
      at[j] = reinterpret_cast<uint64_t*>(PyBytes_AS_STRING(b));
    }
    whole = b != nullptr;
  }
  if (!whole) {
    Py_XDECREF(out); Py_XDECREF(counts);
    return nullptr;
  }
  int64_t* c = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(counts));
  int type = kOther;
  long device = kNone;
  bool plain = true;
  try {
    for (Py_ssize_t i = 0; plain && i < n; ++i) {
      const at::Tensor* t[6];
      for (Py_ssize_t j = 0; plain && j < k; ++j) {
        PyObject* o = PyList_GET_ITEM(l[j], i);
        plain = THPVariable_Check(o);
        if (!plain) break;
        t[j] = &THPVariable_Unpack(o);
        plain = t[j]->is_cuda() && (device == kNone || t[j]->get_device() == device);
        if (plain) device = t[j]->get_device();
      }
      if (!plain) break;
      const at::Tensor& p = *t[0];
      if (i == 0) type = type_code(p);
      plain = type >= kF32 && type <= kF16 && type_code(p) == type && dense(p) && type_code(*t[1]) == type &&
              type_code(*t[2]) == kF32 && t[2]->numel() == 1 && type_code(*t[3]) == moment && type_code(*t[4]) == moment;
      for (int j = 1; plain && j < 5; ++j)
        if (j != 2) plain = t[j]->sizes() == p.sizes() && same_order(p, *t[j]);
      if (plain && k == 6) plain = rows_for(p, *t[5], block);
      if (!plain) break;
      for (Py_ssize_t j = 0; j < k; ++j) at[j][i] = reinterpret_cast<uint64_t>(t[j]->data_ptr());
      c[i] = p.numel();
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    Py_DECREF(out); Py_DECREF(counts);
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "step_lists: unknown C++ exception");
    Py_DECREF(out); Py_DECREF(counts);
    return nullptr;
  }
  if (!plain) {
    Py_DECREF(out); Py_DECREF(counts);
    Py_RETURN_NONE;
  }
  return Py_BuildValue("(ilNN)", type, device, out, counts);
}

// bump(list, ...): the kernels wrote these tensors behind autograd's back; tell it, as torch's own in-place operations do
PyObject* bump(PyObject*, PyObject* args) {
  try {
    for (Py_ssize_t j = 0; j < PyTuple_GET_SIZE(args); ++j) {
      PyObject* list = PyTuple_GET_ITEM(args, j);
      if (!is_list(list, "bump")) return nullptr;
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
        PyObject* o = PyList_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) {
          PyErr_SetString(PyExc_TypeError, "expected tensors");
          return nullptr;
        }
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
      }
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "bump: unknown C++ exception");
    return nullptr;
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"describe", describe, METH_O, "addresses, element counts, types, device, common type, first not dense"},
                         {"differ", differ, METH_VARARGS, "first place where two lists differ in shape or memory order"},
                         {"rows_of", rows_of, METH_VARARGS, "first matrix that has not a row for every block of its tensor"},
                         {"step_lists", step_lists, METH_VARARGS, "the arrays of an optimizer step, or None"},
                         {"bump", bump, METH_VARARGS, "count a version of every tensor"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensorlist", "lists of tensors for multi-tensor calls", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensorlist(void) { return PyModule_Create(&module); }
