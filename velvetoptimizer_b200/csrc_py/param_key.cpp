// Host helpers of the PyTorch layer: the modules' repack check (pairs) and the gradient
// clipping's tensor table (grad_table).  The repack check is the (data pointer, version) pair of
// every parameter of a list in one call, as bytes (16 per tensor).  The modules compare
// these bytes before each forward to see whether the packed weights are stale; done in
// Python, reading 900 parameters' pointers and versions one attribute at a time costs more
// than a decode-sized forward on the GPU.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include <torch/csrc/autograd/python_variable.h>

namespace {

PyObject* pairs(PyObject*, PyObject* seq) {
  PyObject* fast = PySequence_Fast(seq, "pairs() takes a sequence of tensors");
  if (!fast) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
  PyObject* out = PyBytes_FromStringAndSize(nullptr, n * 16);
  if (!out) {
    Py_DECREF(fast);
    return nullptr;
  }
  char* buf = PyBytes_AS_STRING(out);
  PyObject** items = PySequence_Fast_ITEMS(fast);
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_Check(items[i])) {
        PyErr_SetString(PyExc_TypeError, "pairs() takes a sequence of tensors");
        Py_DECREF(out);
        Py_DECREF(fast);
        return nullptr;
      }
      const at::Tensor& t = THPVariable_Unpack(items[i]);
      const uint64_t v[2] = {static_cast<uint64_t>(reinterpret_cast<uintptr_t>(t.data_ptr())),
                             static_cast<uint64_t>(t._version())};
      std::memcpy(buf + 16 * i, v, 16);
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    Py_DECREF(out);
    Py_DECREF(fast);
    return nullptr;
  }
  Py_DECREF(fast);
  return out;
}

// grad_table(tensors, use_grad) -> None when there is no tensor, else (pointers int64, counts
// int64, dtypes int32, as bytes; device index; positions in `tensors` of the ones that are not
// dense and so left out).  The tensors are the sequence's own, or their .grad where present.
// A tensor given twice is taken once; tensors that overlap otherwise, lie on several devices
// or have another type raise.
PyObject* grad_table(PyObject*, PyObject* args) {
  PyObject* seq;
  int use_grad;
  if (!PyArg_ParseTuple(args, "Op", &seq, &use_grad)) return nullptr;
  PyObject* fast = PySequence_Fast(seq, "grad_table() takes a sequence of tensors");
  if (!fast) return nullptr;
  PyObject* odd = nullptr;
  PyObject* result = nullptr;
  struct Entry {
    int64_t ptr, count, bytes;
    int32_t dtype;
  };
  try {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
    PyObject** items = PySequence_Fast_ITEMS(fast);
    std::vector<Entry> table;
    table.reserve(static_cast<size_t>(n));
    int device = -1;
    bool any = false;
    odd = PyList_New(0);
    if (!odd) throw std::bad_alloc();
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_Check(items[i])) {
        PyErr_SetString(PyExc_TypeError, "expected tensors");
        throw 0;
      }
      const at::Tensor& own = THPVariable_Unpack(items[i]);
      const at::Tensor& t = use_grad ? own.grad() : own;
      if (!t.defined()) continue;
      any = true;
      if (t.layout() != at::kStrided) {
        PyErr_SetString(PyExc_TypeError, "sparse gradients are not supported");
        throw 0;
      }
      if (!t.is_cuda()) {
        PyErr_SetString(PyExc_RuntimeError,
                        "gradients must be CUDA tensors (there is no CPU path)");
        throw 0;
      }
      if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) {
        PyErr_SetString(PyExc_TypeError, "gradients must be float32 or bfloat16");
        throw 0;
      }
      const int d = t.device().index();
      if (device >= 0 && d != device) {
        PyErr_SetString(PyExc_ValueError, "gradients must lie on one device");
        throw 0;
      }
      device = d;
      if (t.numel() == 0) continue;
      if (!t.is_non_overlapping_and_dense()) {
        PyObject* k = PyLong_FromSsize_t(i);
        const int rc = k ? PyList_Append(odd, k) : -1;
        Py_XDECREF(k);
        if (rc != 0) throw 0;
        continue;
      }
      Entry e;
      e.ptr = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()));
      e.count = t.numel();
      e.dtype = t.scalar_type() == at::kBFloat16 ? 1 : 0;
      e.bytes = e.count * (e.dtype ? 2 : 4);
      table.push_back(e);
    }
    if (!any) {
      Py_DECREF(odd);
      Py_DECREF(fast);
      Py_RETURN_NONE;
    }
    // by address: a repeated tensor and an overlap are neighbours
    std::vector<size_t> order(table.size());
    for (size_t i = 0; i < order.size(); ++i) order[i] = i;
    std::sort(order.begin(), order.end(), [&](size_t a, size_t b) {
      return table[a].ptr != table[b].ptr ? table[a].ptr < table[b].ptr : a < b;
    });
    std::vector<char> drop(table.size(), 0);
    int64_t end = 0;
    size_t last = 0;
    for (size_t k = 0; k < order.size(); ++k) {
      const Entry& e = table[order[k]];
      if (k > 0 && e.ptr < end) {
        const Entry& p = table[last];
        if (e.ptr == p.ptr && e.bytes == p.bytes && e.dtype == p.dtype) {
          drop[order[k]] = 1;
          continue;
        }
        PyErr_SetString(PyExc_ValueError, "gradients overlap in memory");
        throw 0;
      }
      end = e.ptr + e.bytes;
      last = order[k];
    }
    std::string ptrs, counts, dtypes;
    for (size_t i = 0; i < table.size(); ++i) {
      if (drop[i]) continue;
      ptrs.append(reinterpret_cast<const char*>(&table[i].ptr), 8);
      counts.append(reinterpret_cast<const char*>(&table[i].count), 8);
      dtypes.append(reinterpret_cast<const char*>(&table[i].dtype), 4);
    }
    result = Py_BuildValue("(y#y#y#iO)", ptrs.data(), static_cast<Py_ssize_t>(ptrs.size()),
                           counts.data(), static_cast<Py_ssize_t>(counts.size()), dtypes.data(),
                           static_cast<Py_ssize_t>(dtypes.size()), device, odd);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (int) {  // the Python error is set
  }
  Py_XDECREF(odd);
  Py_DECREF(fast);
  return result;
}

PyMethodDef kMethods[] = {
    {"grad_table", grad_table, METH_VARARGS, "addresses, sizes and types of dense tensors"},
    {"pairs", pairs, METH_O, "(data_ptr, version) of every tensor, 16 bytes each"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_param_key", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__param_key() { return PyModule_Create(&kModule); }
