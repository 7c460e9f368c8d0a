// The short way from the paged operators' Python functions into the library. A decoding step makes these calls once per layer for a few
// microseconds of GPU work each; argument tuples, ctypes conversions and attribute reads made up 10 of a call's 15 us of host time.
//
// A call whose tensors have a layout (types, sizes, strides, device, and the arguments that the checks look at) that the Python side has
// checked before is made from here; any other returns None, and the Python function checks it, makes the call and has its layout
// remembered (`learn`). Nothing of a tensor but its layout is kept.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cstring>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/spinf_b200.h"

namespace {

struct Key {
  std::string bytes;
  int device = -2;  // of the call's tensors (-2: none yet, -1: not one CUDA device)
  void num(int64_t x) { bytes.append(reinterpret_cast<const char*>(&x), 8); }
  // the tensor's layout; null: None
  bool tensor(PyObject* o, const at::Tensor*& t) {
    t = nullptr;
    if (o == Py_None) {
      num(-1);
      return true;
    }
    if (!THPVariable_Check(o)) return false;
    t = &THPVariable_Unpack(o);
    if (!t->is_cuda()) return false;
    const int d = t->get_device();
    if (device == -2) device = d;
    else if (device != d) return false;
    num((static_cast<int64_t>(t->scalar_type()) << 8) | t->dim());
    for (const int64_t x : t->sizes()) num(x);
    for (const int64_t x : t->strides()) num(x);
    return true;
  }
};

using Layouts = std::unordered_map<std::string, std::vector<int64_t>>;
Layouts g_layouts;
constexpr size_t MOST_LAYOUTS = 4096;  // then they are learnt anew: a bound for programs whose sizes never repeat

int64_t number(PyObject* o) { return o == Py_None ? INT64_MIN : PyLong_AsLongLong(o); }
void* data(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// what the functions below share: the key of a call, and its checked layout if there is one
enum { APPEND, ATTENTION, EVICT };
struct Call {
  Key key;
  std::vector<int64_t> layout;  // (a copy: what the call allocates may run other code that learns)
  bool plain = true;  // the arguments are ones that a key can be made of
  void find() {
    if (!plain || PyErr_Occurred()) {
      PyErr_Clear();  // the Python function says what is wrong
      plain = false;
      return;
    }
    const auto it = g_layouts.find(key.bytes);
    if (it != g_layouts.end() && key.device == c10::cuda::current_device()) layout = it->second;
  }
};
constexpr int TENSORS = 10;
// `which`: the operator; args: its tensors first, then what its layout depends on
Call make_call(int which, PyObject* const* args, int tensors, int numbers, const at::Tensor** t) {
  Call c;
  c.key.bytes.reserve(1024);
  c.key.num(which);
  for (int i = 0; i < tensors && c.plain; ++i) c.plain = c.key.tensor(args[i], t[i]);
  if (c.plain) {
    for (int i = 0; i < numbers; ++i) c.key.num(number(args[tensors + i]));
    c.key.num(c.key.device);
  }
  c.find();
  return c;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) { return at::empty(sizes, like.options().dtype(type)); }
bool wrong_count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return n != want;
}

// qkv, k, v, table, lens, cu, wq, wk, cos, sin | H, Hkv, D | eps, plus1, norm_v -> q, None, or an error's number
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (wrong_count(n_args, 16)) return nullptr;
  const at::Tensor* t[TENSORS];
  const Call c = make_call(APPEND, args, 10, 3, t);
  if (c.layout.empty() || data(t[1]) == data(t[2])) Py_RETURN_NONE;
  const int64_t* x = c.layout.data();  // n, pitch, rot, pages, page, k strides, v strides, table pitch, width, B
  const int64_t H = PyLong_AsLongLong(args[10]), h = PyLong_AsLongLong(args[11]), D = PyLong_AsLongLong(args[12]);
  const double eps = PyFloat_AsDouble(args[13]);
  const int plus1 = PyObject_IsTrue(args[14]), norm_v = PyObject_IsTrue(args[15]);
  if (PyErr_Occurred()) return nullptr;
  const bool moved = t[6] || x[2] > 0;
  at::Tensor q = moved ? make({x[0], H, D}, at::kBFloat16, *t[0]) : t[0]->narrow(1, 0, H * D).view({x[0], H, D});
  const int rc = spinf_paged_append(data(t[0]), x[1], x[0], H, h, D, data(t[6]), data(t[7]), x[2] ? data(t[8]) : nullptr, x[2] ? data(t[9]) : nullptr, x[2], eps,
                                    plus1, norm_v, moved ? q.data_ptr() : nullptr, data(t[1]), data(t[2]), x[3], x[4], x + 5, x + 8,
                                    static_cast<int32_t*>(data(t[3])), x[11], x[12], static_cast<int32_t*>(data(t[4])), static_cast<int32_t*>(data(t[5])), x[13],
                                    stream_of(c.key.device));
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(q);
  END_HANDLE_TH_ERRORS
}

// q, k, v, table, lens, cu, weights, weights_out, out, workspace | max_q, window, max_len, shared | scale, decay -> out, None, or an
// error's number. (The workspace is no part of the layout.)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (wrong_count(n_args, 16)) return nullptr;
  const at::Tensor* t[TENSORS] = {};
  PyObject* in[13];
  std::memcpy(in, args, 9 * sizeof(PyObject*));
  std::memcpy(in + 9, args + 10, 4 * sizeof(PyObject*));
  const Call c = make_call(ATTENTION, in, 9, 4, t);
  if (c.layout.empty()) Py_RETURN_NONE;
  if (args[9] != Py_None) {
    if (!THPVariable_Check(args[9])) Py_RETURN_NONE;
    t[9] = &THPVariable_Unpack(args[9]);
    if (!t[9]->is_cuda() || t[9]->get_device() != c.key.device || !t[9]->is_contiguous()) Py_RETURN_NONE;
  }
  // n, H, h, D, q pitch, out pitch, pages, page, k strides, v strides, table pitch, B, max_len, window, workspace, shared, weight strides
  const int64_t* x = c.layout.data();
  if (t[8] && x[0] && data(t[8]) == data(t[0])) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(args[14]), decay = PyFloat_AsDouble(args[15]);
  const int64_t max_q = PyLong_AsLongLong(args[10]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out = t[8] ? *t[8] : make({x[0], x[1], x[3]}, at::kBFloat16, *t[0]), ws;
  void* space = nullptr;
  if (x[18] > 0) {
    if (!t[9] || static_cast<int64_t>(t[9]->nbytes()) < x[18]) ws = make({x[18]}, at::kByte, *t[0]);
    space = ws.defined() ? ws.data_ptr() : t[9]->data_ptr();
  }
  const int rc = spinf_paged_attention(data(t[0]), x[4], x[0], x[1], x[2], x[3], data(t[1]), data(t[2]), x[6], x[7], x + 8, x + 11, static_cast<int32_t*>(data(t[3])),
                                       x[14], static_cast<int32_t*>(data(t[4])), static_cast<int32_t*>(data(t[5])), x[15], max_q, x[16], x[17], x[19], scale,
                                       static_cast<float*>(data(t[6])), static_cast<float*>(data(t[7])), t[6] ? x + 20 : nullptr, decay, out.data_ptr(), x[5], space,
                                       x[18], stream_of(c.key.device));
  return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// k, v, table, lens, weights, new_table | keep, recent, max_len -> (new lens, kept, weights or None), None, or an error's number
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (wrong_count(n_args, 9)) return nullptr;
  const at::Tensor* t[TENSORS];
  const Call c = make_call(EVICT, args, 6, 3, t);
  if (c.layout.empty()) Py_RETURN_NONE;
  const int64_t* x = c.layout.data();  // pages, h, page, D, k strides, v strides, B, table pitch, new pitch, max_len, weight strides, recent
  const int64_t keep = PyLong_AsLongLong(args[6]);
  at::Tensor lens = make({x[10]}, at::kInt, *t[0]), kept = make({x[10], x[1], keep}, at::kInt, *t[0]), w;
  if (t[4]) w = make({x[10], x[1], keep}, at::kFloat, *t[0]);
  const int rc = spinf_paged_evict(data(t[0]), data(t[1]), x[0], x[2], x[1], x[3], x + 4, x + 7, static_cast<int32_t*>(data(t[2])), x[11],
                                   static_cast<int32_t*>(data(t[3])), x[10], x[13], static_cast<float*>(data(t[4])), x[14], x[15], keep, x[16],
                                   static_cast<int32_t*>(data(t[5])), x[12], lens.data_ptr<int32_t>(), kept.data_ptr<int32_t>(), t[4] ? w.data_ptr<float>() : nullptr,
                                   stream_of(c.key.device));
  if (rc) return PyLong_FromLong(rc);
  PyObject* weights = t[4] ? THPVariable_Wrap(w) : Py_NewRef(Py_None);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(lens), THPVariable_Wrap(kept), weights);
  END_HANDLE_TH_ERRORS
}

// kernels that this thread's last call has launched, whichever way it went
PyObject* launches(PyObject*, PyObject*) { return PyLong_FromLongLong(spinf_paged_launches()); }

// (operator, its tensors and the numbers of its key, the checked layout): the next call with this key is made from here
PyObject* learn(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (wrong_count(n_args, 3)) return nullptr;
  const int which = static_cast<int>(PyLong_AsLong(args[0]));
  const int tensors = which == APPEND ? 10 : which == ATTENTION ? 9 : 6, numbers = which == ATTENTION ? 4 : 3;
  if (!PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != tensors + numbers || !PyTuple_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError, "learn: expected an operator's arguments and its layout");
    return nullptr;
  }
  std::vector<PyObject*> in;
  for (int i = 0; i < tensors + numbers; ++i) in.push_back(PyTuple_GET_ITEM(args[1], i));
  const at::Tensor* t[TENSORS];
  const Call c = make_call(which, in.data(), tensors, numbers, t);
  std::vector<int64_t> layout;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[2]); ++i) layout.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(args[2], i)));
  if (PyErr_Occurred()) return nullptr;
  if (c.plain) {
    if (g_layouts.size() >= MOST_LAYOUTS) g_layouts.clear();
    g_layouts[c.key.bytes] = layout;
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef METHODS[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(evict)), METH_FASTCALL, nullptr},
    {"launches", launches, METH_NOARGS, nullptr},
    {"learn", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(learn)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef MODULE = {PyModuleDef_HEAD_INIT, "paged_bind", nullptr, -1, METHODS, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_paged_bind() {
  PyObject* m = PyModule_Create(&MODULE);
  if (m) PyModule_AddStringConstant(m, "made_for", SPINF_MADE_FOR);  // (the loader and the build look at it)
  return m;
}
