// Reads lists of torch tensors into the records of the optimizer entry points (include/oivae_hip.h): addresses, sizes and
// types of parameters and gradients.  In Python this costs about a microsecond a tensor and check, ten checks a tensor --
// more than the kernels of a small model take; here a tensor costs about 20 ns.  Only the ordinary case is served: the
// functions return the index of the first tensor that is anything else (another type, size, device or order than its
// record says), and oi_vae_amd/optim.py then goes through the list itself, copies what can be copied and refuses the rest.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <vector>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/oivae_hip.h"

namespace {

int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return OIVAE_F32;
    case at::kBFloat16: return OIVAE_BF16;
    case at::kHalf: return OIVAE_F16;
    default: return -1;
  }
}

// one piece of device memory on `device`, its values as they stand
bool plain(const at::Tensor& t, int device) {
  return t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && !t.is_neg() && type_of(t) >= 0 &&
         (t.is_contiguous() || t.is_non_overlapping_and_dense());
}

// The order of a dense tensor's elements in memory: 0 row by row, else a number that another order hardly shares (a hash of
// the sizes and strides of the dimensions that have any).  Moments lie in the order their parameter had at first.
int32_t order_of(const at::Tensor& t) {
  if (t.is_contiguous()) return 0;
  uint32_t h = 2166136261u;
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) == 1) continue;
    h = (h ^ (uint32_t)t.size(d)) * 16777619u;
    h = (h ^ (uint32_t)t.stride(d)) * 16777619u;
  }
  return (int32_t)(h | 1u);
}

// what autograd is told where a kernel writes a tensor behind its back: a graph that saved it says so instead of going on
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Buffer {
  Py_buffer b;
  bool held = false;
  ~Buffer() { if (held) PyBuffer_Release(&b); }
  bool take(PyObject* o, Py_ssize_t item, Py_ssize_t count) {
    if (PyObject_GetBuffer(o, &b, PyBUF_WRITABLE | PyBUF_C_CONTIGUOUS) != 0) return false;
    held = true;
    if (b.len < item * count) {
      PyErr_SetString(PyExc_ValueError, "fewer records than tensors");
      return false;
    }
    return true;
  }
};

// parameters(list, records of oivae_adamw_tensor_t, device, records of oivae_grad_t or None) -> (first unusual tensor or -1,
// number without a gradient).  Fills p, g and g_type, g = 0 where a parameter has no gradient (an address that nothing reads
// where it has one without elements, whose own is 0), and the gradients' records (n = 0 and index -1 there).  The records' n,
// p_type and pad (the order of its elements) say what the parameters have to be.
PyObject* parameters(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4 || !PyList_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "parameters(list, records, device, gradient records)");
    return nullptr;
  }
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  Buffer buf, gbuf;
  if (!buf.take(args[1], sizeof(oivae_adamw_tensor_t), n)) return nullptr;
  const long device = PyLong_AsLong(args[2]);
  if (device == -1 && PyErr_Occurred()) return nullptr;
  if (args[3] != Py_None && !gbuf.take(args[3], sizeof(oivae_grad_t), n)) return nullptr;
  oivae_adamw_tensor_t* r = static_cast<oivae_adamw_tensor_t*>(buf.b.buf);
  oivae_grad_t* q = gbuf.held ? static_cast<oivae_grad_t*>(gbuf.b.buf) : nullptr;
  long missing = 0;
  Py_ssize_t unusual = -1;
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(args[0], i);
      unusual = i;
      if (!THPVariable_Check(o)) break;
      const at::Tensor& p = THPVariable_Unpack(o);
      const at::Tensor& g = p.grad();
      if (!g.defined()) {
        r[i].g = nullptr;
        if (q) q[i] = oivae_grad_t{nullptr, 0, OIVAE_F32, -1};
        ++missing;
        unusual = -1;
        continue;
      }
      if (!plain(p, (int)device) || !plain(g, (int)device) || p.numel() != r[i].n || type_of(p) != r[i].p_type || !g.sizes().equals(p.sizes()))
        break;
      const bool rows = p.is_contiguous();
      if (!(rows && g.is_contiguous()) && !g.strides().equals(p.strides())) break;
      if ((rows ? 0 : order_of(p)) != r[i].pad) break;
      written(p);
      r[i].p = p.data_ptr();
      r[i].g = g.numel() > 0 ? g.data_ptr() : reinterpret_cast<void*>(16);
      r[i].g_type = type_of(g);
      if (q) q[i] = oivae_grad_t{g.data_ptr(), g.numel(), type_of(g), r[i].index};
      unusual = -1;
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return Py_BuildValue("(nl)", unusual, missing);
}

// gradients(list, records of oivae_grad_t, whether they will be written) -> (count, device, address of the
// records) of the gradients that are there, or None when one is unusual, shares memory with another (or appears twice) or is
// on another device; (0, -1, address) without any.
PyObject* gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3 || !PyList_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "gradients(list, records, written)");
    return nullptr;
  }
  const Py_ssize_t n = PyList_GET_SIZE(args[0]);
  const bool write = args[2] == Py_True;
  Buffer buf;
  if (!buf.take(args[1], sizeof(oivae_grad_t), n)) return nullptr;
  oivae_grad_t* r = static_cast<oivae_grad_t*>(buf.b.buf);
  long count = 0;
  int device = -1;
  try {
    struct Span { const char *begin, *end; };
    std::vector<Span> seen;
    seen.reserve((size_t)n);
    bool ascending = true;   // as the parts of one buffer are; a sort of 65 spans takes a microsecond
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(args[0], i);
      if (!THPVariable_Check(o)) Py_RETURN_NONE;
      const at::Tensor& g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      if (device < 0 && g.is_cuda()) device = (int)g.get_device();
      if (!plain(g, device)) Py_RETURN_NONE;
      r[count++] = oivae_grad_t{g.data_ptr(), g.numel(), type_of(g), -1};
      if (g.numel() > 0) {
        const char* at = static_cast<const char*>(g.data_ptr());
        if (!seen.empty() && at < seen.back().end) ascending = false;
        seen.push_back(Span{at, at + g.numel() * (type_of(g) == OIVAE_F32 ? 4 : 2)});
      }
    }
    if (!ascending) {
      std::sort(seen.begin(), seen.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
      for (size_t i = 1; i < seen.size(); ++i)
        if (seen[i].begin < seen[i - 1].end) Py_RETURN_NONE;
    }
    for (Py_ssize_t i = 0; write && i < n; ++i) {
      const at::Tensor& g = THPVariable_Unpack(PyList_GET_ITEM(args[0], i)).grad();
      if (g.defined()) written(g);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return Py_BuildValue("(liK)", count, device, (unsigned long long)reinterpret_cast<uintptr_t>(r));
}

// order(tensor) -> order_of
PyObject* order(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 1 || !THPVariable_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "order(tensor)");
    return nullptr;
  }
  try {
    return PyLong_FromLong(order_of(THPVariable_Unpack(args[0])));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"order", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(order)), METH_FASTCALL, nullptr},
    {"parameters", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(parameters)), METH_FASTCALL, nullptr},
    {"gradients", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gradients)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists(void) { return PyModule_Create(&module); }
