// Host only: reads lists of tensors for the optimizer's calls (ganet_amd/optim.py).
//
// A step checks every tensor of every list (GPU, type, shape, order, address): in Python that is
// some 40 ns an attribute, 100 us for the seven lists of a 62-tensor model, as long as the step
// itself.  Here it is a few.  Both functions only accept the plain case - one GPU, one type a list,
// everything contiguous and of its parameter's shape, nothing twice - and return None for anything
// else; Python then looks again, copies what can be copied and names what is wrong.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <vector>

namespace {

enum { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2, kE4M3 = 3, kOther = -1 };

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return kFloat32;
    case at::kBFloat16: return kBFloat16;
    case at::kHalf: return kFloat16;
    case at::kFloat8_e4m3fn: return kE4M3;
    default: return kOther;
  }
}

// The i-th tensor of a list or tuple, null where it is none.
const at::Tensor *item(PyObject *list, Py_ssize_t i) {
  PyObject *o = PyList_Check(list) ? PyList_GET_ITEM(list, i) : PyTuple_GET_ITEM(list, i);
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}
Py_ssize_t length(PyObject *list) {
  if (PyList_Check(list)) return PyList_GET_SIZE(list);
  return PyTuple_Check(list) ? PyTuple_GET_SIZE(list) : -1;
}

PyObject *bytes(const void *p, size_t n) {
  return PyBytes_FromStringAndSize(static_cast<const char *>(p), static_cast<Py_ssize_t>(n));
}

// step(params, grads, avgs, seconds, avg_scales, second_scales, masters, block) ->
// (gpu, parameter type, gradient type, state type, rows of ganet_step_tensor) or None
PyObject *step(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "step() takes 8 arguments");
    return nullptr;
  }
  const long block = PyLong_AsLong(args[7]);
  if (block < 1) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "step(): block");
    return nullptr;
  }
  try {
    const Py_ssize_t n = length(args[0]);
    if (n < 1) Py_RETURN_NONE;
    std::vector<std::uint64_t> rows(static_cast<size_t>(n) * 8, 0);
    std::vector<std::uint64_t> written;
    int types[7] = {kOther, kOther, kOther, kOther, kOther, kOther, kOther};
    int gpu = -1;
    for (int k = 0; k < 7; ++k) {
      if (args[k] == Py_None) {
        if (k < 4) Py_RETURN_NONE;
        continue;
      }
      if (length(args[k]) != n) Py_RETURN_NONE;
      for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor *t = item(args[k], i), *p = item(args[0], i);
        if (!t || !p || !t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous()) Py_RETURN_NONE;
        const int type = code(t->scalar_type()), at = static_cast<int>(t->get_device());
        if (i == 0) types[k] = type;
        if (i == 0 && k == 0) gpu = at;
        if (type == kOther || type != types[k] || at != gpu) Py_RETURN_NONE;
        const std::int64_t values = p->numel();
        if (k == 4 || k == 5) {
          if (t->numel() != (values + block - 1) / block) Py_RETURN_NONE;
        } else if (!t->sizes().equals(p->sizes())) {
          Py_RETURN_NONE;
        }
        const auto address = reinterpret_cast<std::uint64_t>(t->data_ptr());
        rows[i * 8 + k] = address;
        if (k == 0) rows[i * 8 + 7] = static_cast<std::uint64_t>(values);
        if (k != 1 && values) written.push_back(address);
      }
    }
    std::sort(written.begin(), written.end());
    if (std::adjacent_find(written.begin(), written.end()) != written.end()) Py_RETURN_NONE;
    if (types[2] != types[3] || (args[6] != Py_None && types[6] != kFloat32)) Py_RETURN_NONE;
    for (int k = 4; k < 6; ++k)
      if ((args[k] == Py_None) != (types[2] != kE4M3) || (args[k] != Py_None && types[k] != kFloat32))
        Py_RETURN_NONE;
    return Py_BuildValue("iiiiN", gpu, types[0], types[1], types[2], bytes(rows.data(), rows.size() * 8));
  } catch (const std::exception &) {   // a tensor without storage: Python's own reading names it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// grads(list) -> (gpu, addresses, sizes, types) or None
PyObject *grads(PyObject *, PyObject *list) {
  try {
    const Py_ssize_t n = length(list);
    if (n < 1) Py_RETURN_NONE;
    std::vector<std::uint64_t> address(n);
    std::vector<std::int64_t> size(n);
    std::vector<std::int32_t> type(n);
    int gpu = -1;
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor *t = item(list, i);
      if (!t || !t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous()) Py_RETURN_NONE;
      type[i] = code(t->scalar_type());
      if (i == 0) gpu = static_cast<int>(t->get_device());
      if (type[i] == kOther || type[i] == kE4M3 || t->get_device() != gpu) Py_RETURN_NONE;
      address[i] = reinterpret_cast<std::uint64_t>(t->data_ptr());
      size[i] = t->numel();
    }
    return Py_BuildValue("iNNN", gpu, bytes(address.data(), n * 8), bytes(size.data(), n * 8),
                         bytes(type.data(), n * 4));
  } catch (const std::exception &) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

PyMethodDef methods[] = {
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(step)), METH_FASTCALL,
     "The table of an AdamW step over plain lists of tensors, or None."},
    {"grads", grads, METH_O, "Addresses, sizes and types of a plain list of gradients, or None."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_lists", "Reads lists of tensors at C speed.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_lists(void) { return PyModule_Create(&module); }
