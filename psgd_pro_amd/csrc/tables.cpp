// The host tables of an AdamW step from Python's lists of tensors: a Python module of its own, since reading a tensor's address,
// size and type through the interpreter costs some 80 ns each (193 tensors with their gradients and states: 300 us).
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>

#include <sstream>
#include <vector>

namespace {

constexpr int kVersion = 2;      // of these functions and of the layout of what they fill: the bindings ask for their own (_lib.py)
constexpr int64_t kBlock = 256;  // elements that share a scale

struct Fail {
  PyObject* kind;
  std::string text;
};
template <typename... A>
[[noreturn]] void refuse(PyObject* kind, const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Fail{kind, s.str()};
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
std::string what(PyObject* o) {
  std::ostringstream s;
  const at::Tensor* t = tensor(o);
  if (t) s << "one of " << t->sizes() << " in " << t->dtype() << " on " << t->device();
  else s << Py_TYPE(o)->tp_name;
  return s.str();
}

// Addresses, none of them null: a table at most half full (a set with a node for each takes a fifth of the step's host time).
class Seen {
  std::vector<const void*> at_;
  int shift_ = 60;

 public:
  explicit Seen(size_t most) {
    while ((size_t)1 << (64 - shift_) < 2 * most) --shift_;
    at_.resize((size_t)1 << (64 - shift_));
  }
  bool add(const void* p) {  // false: it is there
    size_t i = (uint64_t)(uintptr_t)p * 0x9E3779B97F4A7C15ull >> shift_;
    for (; at_[i]; i = (i + 1) & (at_.size() - 1))
      if (at_[i] == p) return false;
    at_[i] = p;
    return true;
  }
};

// One state tensor's address: `size` elements of `type` on p's device, contiguous.
void* state(PyObject* o, const at::Tensor& p, at::ScalarType type, int64_t size, const char* name, Py_ssize_t i) {
  const at::Tensor* t = tensor(o);
  if (!t || t->scalar_type() != type || t->numel() != size || t->device() != p.device() || !t->is_contiguous())
    refuse(PyExc_RuntimeError, name, " ", i, ": ", size, " elements in ", type, " on ", p.device(), ", contiguous, expected; got ",
           what(o));
  return t->data_ptr();
}

// adamw(params, grads, exp_avgs, exp_avg_sqs, address, count): fills the `count` int64 at `address`, 8 a parameter, array by array:
// elements, dtype (two 32-bit numbers each, the first half), the addresses of parameters, gradients, first moments, second moments
// and their scales. Returns (bits of the states, the gradients that were copied to be contiguous).
PyObject* adamw(PyObject*, PyObject* args) {
  PyObject *params, *grads, *ms, *vs;
  unsigned long long address;
  Py_ssize_t count;
  if (!PyArg_ParseTuple(args, "O!O!O!O!Kn", &PyList_Type, &params, &PyList_Type, &grads, &PyList_Type, &ms, &PyList_Type, &vs, &address,
                        &count))
    return nullptr;
  HANDLE_TH_ERRORS
  try {
    const Py_ssize_t n = PyList_GET_SIZE(params);
    if (!n) refuse(PyExc_RuntimeError, "no parameters");
    if (PyList_GET_SIZE(grads) != n) refuse(PyExc_RuntimeError, PyList_GET_SIZE(grads), " gradients for ", n, " parameters");
    if (PyList_GET_SIZE(ms) != n) refuse(PyExc_RuntimeError, PyList_GET_SIZE(ms), " exp_avgs for ", n, " parameters");
    if (PyList_GET_SIZE(vs) != n) refuse(PyExc_RuntimeError, PyList_GET_SIZE(vs), " exp_avg_sqs for ", n, " parameters");
    if (count != 8 * n) refuse(PyExc_RuntimeError, "a buffer of ", 8 * n, " numbers expected, got one of ", count);
    int64_t* const numel = reinterpret_cast<int64_t*>(address);
    int32_t* const dtype = reinterpret_cast<int32_t*>(numel + n);
    void** const at = reinterpret_cast<void**>(numel + 2 * n);
    const bool pair = PyTuple_Check(PyList_GET_ITEM(ms, 0)) || PyList_Check(PyList_GET_ITEM(ms, 0));
    Seen seen(5 * n);
    std::vector<at::Tensor> copies;
    c10::Device device(c10::kCPU);
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor* p = tensor(PyList_GET_ITEM(params, i));
      if (p && i == 0) device = p->device();
      if (!p || !p->is_cuda() || p->device() != device)
        refuse(PyExc_RuntimeError, "parameter ", i, ": CUDA (HIP) tensors on one device expected; got ", what(PyList_GET_ITEM(params, i)));
      if (p->scalar_type() != at::kFloat && p->scalar_type() != at::kBFloat16)
        refuse(PyExc_TypeError, "parameter ", i, ": float32 or bfloat16 expected, got ", p->dtype());
      if (!p->is_contiguous()) refuse(PyExc_RuntimeError, "parameter ", i, ": contiguous storage expected, its strides are ", p->strides());
      const int64_t size = p->numel();
      if (size && !seen.add(p->data_ptr())) refuse(PyExc_RuntimeError, "parameter ", i, " is there twice");
      const at::Tensor* g = tensor(PyList_GET_ITEM(grads, i));
      if (!g || g->sizes() != p->sizes() || g->scalar_type() != p->scalar_type() || g->device() != device)
        refuse(PyExc_RuntimeError, "gradient ", i, ": as its parameter, ", p->sizes(), " in ", p->dtype(), " on ", device,
               ", expected; got ", what(PyList_GET_ITEM(grads, i)));
      numel[i] = size;
      dtype[i] = p->scalar_type() == at::kFloat ? 0 : 1;
      at[i] = p->data_ptr();
      if (g->is_contiguous()) {
        at[n + i] = g->data_ptr();
      } else {
        copies.push_back(g->contiguous());
        at[n + i] = copies.back().data_ptr();
      }
      for (int k = 0; k < 2; ++k) {
        PyObject* const s = PyList_GET_ITEM(k ? vs : ms, i);
        const char* const name = k ? "exp_avg_sqs" : "exp_avgs";
        const bool two = PyTuple_Check(s) || PyList_Check(s);
        if (two != pair) refuse(PyExc_RuntimeError, name, " ", i, ": states of 32 and of 8 bits in one call");
        if (!pair) {
          at[(2 + k) * n + i] = state(s, *p, at::kFloat, size, name, i);
          continue;
        }
        if (PySequence_Fast_GET_SIZE(s) != 2) refuse(PyExc_RuntimeError, name, " ", i, ": (codes, scales) expected");
        PyObject** const parts = PySequence_Fast_ITEMS(s);
        at[(2 + k) * n + i] = state(parts[0], *p, at::ScalarType::Float8_e4m3fn, size, name, i);
        at[(4 + k) * n + i] = state(parts[1], *p, at::ScalarType::Float8_e8m0fnu, (size + kBlock - 1) / kBlock, name, i);
      }
      // (a state of two parameters, or of both moments, would be written twice in no order)
      for (int k = 2; k < (pair ? 6 : 4) && size; ++k)
        if (!seen.add(at[k * n + i])) refuse(PyExc_RuntimeError, "a state of parameter ", i, " is there twice");
    }
    PyObject* const kept = PyList_New((Py_ssize_t)copies.size());
    if (!kept) return nullptr;
    for (size_t i = 0; i < copies.size(); ++i) PyList_SET_ITEM(kept, (Py_ssize_t)i, THPVariable_Wrap(copies[i]));
    return Py_BuildValue("iN", pair ? 8 : 32, kept);
  } catch (const Fail& f) {
    PyErr_SetString(f.kind, f.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// changed(params): they count as changed in place, as by torch's own operations.
PyObject* changed(PyObject*, PyObject* params) {
  HANDLE_TH_ERRORS
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
    const at::Tensor& p = *tensor(PyList_GET_ITEM(params, i));
    if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"adamw", adamw, METH_VARARGS, nullptr}, {"changed", changed, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tables", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tables() {
  PyObject* const m = PyModule_Create(&module);
  if (m && PyModule_AddIntConstant(m, "VERSION", kVersion) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
