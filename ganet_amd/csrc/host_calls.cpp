// Host only: the plain case of the training operators' calls (ganet_amd/optim.py, norm.py) without
// Python in between.
//
// A step checks every tensor of every list (GPU, type, shape, order, address): in Python that is
// some 40 ns an attribute, 100 us for the seven lists of a 62-tensor model, as long as the step
// itself.  Here it is a few.  The functions only accept the plain case - one GPU, one type a list,
// everything contiguous and of its parameter's shape, no memory twice - and return None for anything
// else; Python then looks again, copies what can be copied and names what is wrong.
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <utility>
#include <vector>

#include "ganet_hip.h"

namespace {

static_assert(sizeof(ganet_step_tensor) == 64, "eight words a tensor");

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

// The exception under way as Python's (torch.OutOfMemoryError stays one).
PyObject *raised() {
  torch::translate_exception_to_python(std::current_exception());
  return nullptr;
}

PyObject *bytes(const void *p, size_t n) {
  return PyBytes_FromStringAndSize(static_cast<const char *>(p), static_cast<Py_ssize_t>(n));
}

// The table of an AdamW step over the lists params, grads, avgs, seconds, avg_scales, second_scales and
// masters (the last three may be None).
struct Step {
  int gpu, param, grad, state;
  std::vector<std::uint64_t> rows;                   // of ganet_step_tensor
};
bool read(PyObject *const *lists, std::int64_t block, Step &s) {
  const Py_ssize_t n = length(lists[0]);
  if (n < 1) return false;
  s.rows.assign(static_cast<size_t>(n) * 8, 0);
  std::vector<std::pair<std::uint64_t, std::uint64_t>> written;        // addresses and bytes
  int types[7] = {kOther, kOther, kOther, kOther, kOther, kOther, kOther};
  s.gpu = -1;
  for (int k = 0; k < 7; ++k) {
    if (lists[k] == Py_None) {
      if (k < 4) return false;
      continue;
    }
    if (length(lists[k]) != n) return false;
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor *t = item(lists[k], i), *p = item(lists[0], i);
      if (!t || !p || !t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous()) return false;
      const int type = code(t->scalar_type()), at = static_cast<int>(t->get_device());
      if (i == 0) types[k] = type;
      if (i == 0 && k == 0) s.gpu = at;
      if (type == kOther || type != types[k] || at != s.gpu) return false;
      const std::int64_t values = p->numel();
      if (k == 4 || k == 5) {
        if (t->numel() != (values + block - 1) / block) return false;
      } else if (!t->sizes().equals(p->sizes())) {
        return false;
      }
      const auto address = reinterpret_cast<std::uint64_t>(t->data_ptr());
      s.rows[i * 8 + k] = address;
      if (k == 0) s.rows[i * 8 + 7] = static_cast<std::uint64_t>(values);
      if (k != 1 && values) written.emplace_back(address, t->nbytes());
    }
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].first + written[i - 1].second) return false;
  s.param = types[0];
  s.grad = types[1];
  s.state = types[2];
  if (types[2] != types[3] || (types[2] != kFloat32 && types[2] != kE4M3) || types[0] == kE4M3 || types[1] == kE4M3)
    return false;
  if (lists[6] != Py_None && (types[6] != kFloat32 || types[0] == kFloat32)) return false;
  for (int k = 4; k < 6; ++k)
    if ((lists[k] == Py_None) != (types[2] != kE4M3) || (lists[k] != Py_None && types[k] != kFloat32)) return false;
  return true;
}

// The tensors' values have changed: autograd refuses a backward pass that saved the old ones, as it does
// after torch's own in-place operations.
void mark(PyObject *list) {
  for (Py_ssize_t i = 0, n = length(list); i < n; ++i) {
    const at::Tensor *t = item(list, i);
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();   // those have no versions
  }
}

// step(params, grads, avgs, seconds, avg_scales, second_scales, masters, block) ->
// (gpu, parameter type, gradient type, state bits, rows of ganet_step_tensor) or None
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
    Step s;
    if (!read(args, block, s)) Py_RETURN_NONE;
    return Py_BuildValue("iiiiN", s.gpu, s.param, s.grad, s.state == kE4M3 ? 8 : 32, bytes(s.rows.data(), s.rows.size() * 8));
  } catch (...) {   // a tensor without storage: Python's own reading names it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

void *address(PyObject *o) { return PyLong_AsVoidPtr(o); }

// adamw(entry point, the seven lists, block, state bits, step, lr, beta1, beta2, eps, weight_decay,
// grad_stats, skip_nonfinite, seed, gpu, stream) -> the entry point's status, or None where nothing was done
PyObject *adamw(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 21) {
    PyErr_SetString(PyExc_TypeError, "adamw() takes 21 arguments");
    return nullptr;
  }
  auto entry = reinterpret_cast<decltype(&ganet_adamw_step)>(address(args[0]));
  const long block = PyLong_AsLong(args[8]), bits = PyLong_AsLong(args[9]), gpu = PyLong_AsLong(args[19]);
  ganet_adamw_params p = {};
  p.step = PyLong_AsLongLong(args[10]);
  p.lr = PyFloat_AsDouble(args[11]);
  p.beta1 = PyFloat_AsDouble(args[12]);
  p.beta2 = PyFloat_AsDouble(args[13]);
  p.eps = PyFloat_AsDouble(args[14]);
  p.weight_decay = PyFloat_AsDouble(args[15]);
  p.skip_nonfinite = PyObject_IsTrue(args[17]);
  p.seed = static_cast<std::uint32_t>(PyLong_AsUnsignedLongMask(args[18]));
  void *stream = address(args[20]);
  if (PyErr_Occurred()) return nullptr;
  try {
    Step s;
    if (!entry || block < 1 || !read(args + 1, block, s) || s.gpu != gpu || bits != (s.state == kE4M3 ? 8 : 32) ||
        s.rows.size() / 8 > INT32_MAX)
      Py_RETURN_NONE;
    if (args[16] != Py_None) {
      const at::Tensor *t = THPVariable_Check(args[16]) ? &THPVariable_Unpack(args[16]) : nullptr;
      if (!t || !t->is_cuda() || t->get_device() != s.gpu || t->scalar_type() != at::kFloat || t->numel() != 4 ||
          !t->is_contiguous())
        Py_RETURN_NONE;
      p.grad_stats = t->data_ptr<float>();
    }
    p.param_dtype = s.param;
    p.grad_dtype = s.grad;
    p.state_bits = static_cast<std::int32_t>(bits);
    const int rc = entry(reinterpret_cast<const ganet_step_tensor *>(s.rows.data()), static_cast<int>(s.rows.size() / 8),
                         &p, stream);
    if (rc == 0) {
      mark(args[1]);
      if (args[7] != Py_None) mark(args[7]);
    }
    return PyLong_FromLong(rc);
  } catch (...) {
    return raised();
  }
}

// written(list)
PyObject *written(PyObject *, PyObject *list) {
  try {
    mark(list);
    Py_RETURN_NONE;
  } catch (...) {
    return raised();
  }
}

// Addresses, sizes and types of a list of gradients that are all contiguous and on one GPU.
struct Grads {
  std::vector<const void *> address;
  std::vector<std::int64_t> size;
  std::vector<std::int32_t> type;
  int gpu = -1;
};
bool read(PyObject *list, Grads &g) {
  const Py_ssize_t n = length(list);
  if (n < 1) return false;
  g.address.resize(n);
  g.size.resize(n);
  g.type.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor *t = item(list, i);
    if (!t || !t->is_cuda() || t->layout() != at::kStrided || !t->is_contiguous()) return false;
    g.type[i] = code(t->scalar_type());
    if (i == 0) g.gpu = static_cast<int>(t->get_device());
    if (g.type[i] == kOther || g.type[i] == kE4M3 || t->get_device() != g.gpu) return false;
    g.address[i] = t->data_ptr();
    g.size[i] = t->numel();
  }
  return true;
}

// grads(list) -> (gpu, addresses, sizes, types) or None
PyObject *grads(PyObject *, PyObject *list) {
  try {
    Grads g;
    if (!read(list, g)) Py_RETURN_NONE;
    const size_t n = g.size.size();
    return Py_BuildValue("iNNN", g.gpu, bytes(g.address.data(), n * 8), bytes(g.size.data(), n * 8),
                         bytes(g.type.data(), n * 4));
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// ---- layer norm -----------------------------------------------------------------------------
// The calls of ganet_amd/norm.py where tensors lie as the kernels take them: in Python the outputs,
// the parameters and the checks of a small call cost more than its kernel.

struct Where {        // how a tensor's channels lie in memory
  std::int64_t outer, inner, channels;
  bool channels_last;
};

// False where the order is another than rows, an NCHW map or a channels_last one.
bool place(const at::Tensor &x, std::int64_t dim, Where &w) {
  const std::int64_t dims = x.dim();
  if (dim < 0) dim += dims;
  if (dim < 0 || dim >= dims || x.numel() == 0) return false;
  w.channels = x.size(dim);
  w.channels_last = false;
  w.inner = 1;
  if (x.is_contiguous()) {
    for (std::int64_t d = dim + 1; d < dims; ++d) w.inner *= x.size(d);
  } else if (dims == 4 && dim == 1 && x.is_contiguous(at::MemoryFormat::ChannelsLast)) {
    w.channels_last = true;
  } else {
    return false;
  }
  w.outer = x.numel() / w.channels / w.inner;
  return true;
}
bool like(const at::Tensor &t, const at::Tensor &x, const Where &w) {
  if (!t.is_cuda() || t.get_device() != x.get_device() || t.scalar_type() != x.scalar_type() ||
      !t.sizes().equals(x.sizes()))
    return false;
  return w.channels_last ? t.is_contiguous(at::MemoryFormat::ChannelsLast) : t.is_contiguous();
}
const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
// A weight or None: false where it is neither or not [channels] on x's GPU.
bool weight(PyObject *o, const at::Tensor &x, const Where &w, const at::Tensor *&t, int &type) {
  t = nullptr;
  if (o == Py_None) return true;
  t = tensor(o);
  if (!t || !t->is_cuda() || t->get_device() != x.get_device() || t->dim() != 1 || t->numel() != w.channels ||
      !t->is_contiguous())
    return false;
  const int c = code(t->scalar_type());
  if (c == kOther || c == kE4M3 || (type != kOther && c != type)) return false;
  type = c;
  return true;
}
at::Tensor empty_like(const at::Tensor &x, const Where &w) {
  return at::empty(x.sizes(), x.options().requires_grad(false),
                   w.channels_last ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous);
}
ganet_layer_norm_params parameters(const Where &w, int type, int weight_type, float eps) {
  ganet_layer_norm_params p = {};
  p.outer = w.outer;
  p.inner = w.inner;
  p.x_stride = p.y_stride = p.g_stride = w.channels * w.inner;
  p.C = static_cast<std::int32_t>(w.channels);
  p.dtype = type;
  p.weight_dtype = weight_type;
  p.eps = eps;
  return p;
}
void *data(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
PyObject *wrapped(const at::Tensor &t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// grad_norm(workspace query, entry point, gradients, max_norm, inv_scale, gpu, stream) -> the float32 [4]
// tensor, the entry point's status where it is not 0, or None
PyObject *grad_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 7) {
    PyErr_SetString(PyExc_TypeError, "grad_norm() takes 7 arguments");
    return nullptr;
  }
  auto query = reinterpret_cast<decltype(&ganet_grad_norm_workspace_bytes)>(address(args[0]));
  auto entry = reinterpret_cast<decltype(&ganet_grad_norm)>(address(args[1]));
  const double max_norm = PyFloat_AsDouble(args[3]), inv_scale = PyFloat_AsDouble(args[4]);
  const long gpu = PyLong_AsLong(args[5]);
  void *stream = address(args[6]);
  if (PyErr_Occurred()) return nullptr;
  try {
    Grads g;
    if (!query || !entry || !read(args[2], g) || g.gpu != gpu || g.size.size() > 1 << 20) Py_RETURN_NONE;
    const int n = static_cast<int>(g.size.size());
    const auto plain = item(args[2], 0)->options().requires_grad(false);
    const size_t bytes = query(g.size.data(), n);
    const at::Tensor out = at::empty({4}, plain.dtype(at::kFloat));
    const at::Tensor ws = at::empty({static_cast<std::int64_t>(std::max<size_t>(bytes, 256))}, plain.dtype(at::kByte));
    const int rc = entry(g.address.data(), g.size.data(), g.type.data(), n, max_norm, inv_scale, out.data_ptr<float>(),
                         ws.data_ptr(), bytes, stream);
    if (rc) return PyLong_FromLong(rc);
    return wrapped(out);
  } catch (...) {
    return raised();
  }
}

// layer_norm_forward(entry point, x, weight, bias, eps, channel_dim, stats, stream) ->
// (y, mean, rstd), the entry point's status where it is not 0, or None
PyObject *layer_norm_forward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 8) {
    PyErr_SetString(PyExc_TypeError, "layer_norm_forward() takes 8 arguments");
    return nullptr;
  }
  const double eps = PyFloat_AsDouble(args[4]);
  const long dim = PyLong_AsLong(args[5]);
  const int stats = PyObject_IsTrue(args[6]);
  auto entry = reinterpret_cast<decltype(&ganet_layer_norm_forward)>(address(args[0]));
  void *stream = address(args[7]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor *x = tensor(args[1]), *w, *b;
    Where at;
    int weight_type = kOther;
    if (!x || !x->is_cuda() || !entry || !place(*x, dim, at) || at.channels > INT32_MAX) Py_RETURN_NONE;
    const int type = code(x->scalar_type());
    if (type == kOther || type == kE4M3 || !weight(args[2], *x, at, w, weight_type) ||
        !weight(args[3], *x, at, b, weight_type))
      Py_RETURN_NONE;
    const auto p = parameters(at, type, weight_type == kOther ? type : weight_type, static_cast<float>(eps));
    const at::Tensor y = empty_like(*x, at);
    at::Tensor mean, rstd;
    if (stats) {
      mean = at::empty({at.outer * at.inner}, x->options().dtype(at::kFloat).requires_grad(false));
      rstd = at::empty_like(mean);
    }
    const int rc = entry(data(x), data(w), data(b), y.data_ptr(),
                         stats ? mean.data_ptr<float>() : nullptr, stats ? rstd.data_ptr<float>() : nullptr, &p, stream);
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("NNN", wrapped(y), wrapped(mean), wrapped(rstd));
  } catch (...) {
    return raised();
  }
}

// layer_norm_backward(workspace query, entry point, x, weight, grad, mean, rstd, channel_dim,
// need_input + 2 need_weight + 4 need_bias, stream) -> (grad_x, grad_weight, grad_bias), a status, or None
PyObject *layer_norm_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  if (nargs != 10) {
    PyErr_SetString(PyExc_TypeError, "layer_norm_backward() takes 10 arguments");
    return nullptr;
  }
  auto query = reinterpret_cast<decltype(&ganet_layer_norm_backward_workspace_bytes)>(address(args[0]));
  auto entry = reinterpret_cast<decltype(&ganet_layer_norm_backward)>(address(args[1]));
  const long dim = PyLong_AsLong(args[7]), need = PyLong_AsLong(args[8]);
  void *stream = address(args[9]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor *x = tensor(args[2]), *g = tensor(args[4]), *mean = tensor(args[5]), *rstd = tensor(args[6]), *w;
    Where at;
    int weight_type = kOther;
    if (!x || !g || !mean || !rstd || !x->is_cuda() || !query || !entry || need < 1 || need > 7 ||
        !place(*x, dim, at) || at.channels > INT32_MAX || !like(*g, *x, at))
      Py_RETURN_NONE;
    const int type = code(x->scalar_type());
    if (type == kOther || type == kE4M3 || !weight(args[3], *x, at, w, weight_type)) Py_RETURN_NONE;
    for (const at::Tensor *t : {mean, rstd})
      if (!t->is_cuda() || t->get_device() != x->get_device() || t->scalar_type() != at::kFloat ||
          t->numel() != at.outer * at.inner || !t->is_contiguous())
        Py_RETURN_NONE;
    if (weight_type == kOther) weight_type = type;
    const auto p = parameters(at, type, weight_type, 0.0f);
    const auto plain = (w ? w : x)->options().requires_grad(false);
    at::Tensor gx, gw, gb, ws;
    size_t bytes = 0;
    if (need & 1) gx = empty_like(*x, at);
    if (need & 2) gw = at::empty({at.channels}, plain);
    if (need & 4) gb = at::empty({at.channels}, plain);
    if (need & 6) {
      bytes = query(&p);
      ws = at::empty({static_cast<std::int64_t>(std::max<size_t>(bytes, 256))}, plain.dtype(at::kByte));
    }
    auto out = [](const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    const int rc = entry(data(x), data(w), data(g), mean->data_ptr<float>(), rstd->data_ptr<float>(), out(gx), out(gw),
                         out(gb), &p, out(ws), bytes, stream);
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("NNN", wrapped(gx), wrapped(gw), wrapped(gb));
  } catch (...) {
    return raised();
  }
}

PyMethodDef methods[] = {
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(step)), METH_FASTCALL,
     "The table of an AdamW step over plain lists of tensors, or None."},
    {"adamw", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw)), METH_FASTCALL,
     "An AdamW step over plain lists of tensors, or None."},
    {"grads", grads, METH_O, "Addresses, sizes and types of a plain list of gradients, or None."},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_norm)), METH_FASTCALL,
     "The norm of a plain list of gradients, or None."},
    {"written", written, METH_O, "Marks a list of tensors as changed in place."},
    {"layer_norm_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_forward)),
     METH_FASTCALL, "Layer norm's forward on tensors in the kernels' order, or None."},
    {"layer_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(layer_norm_backward)),
     METH_FASTCALL, "Layer norm's backward on tensors in the kernels' order, or None."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Reads lists of tensors at C speed.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
