// The table of a model's gradients (scao_tensor_desc), read from the tensors
// themselves: a model has hundreds of them, and reading six properties of each
// from Python takes longer than the kernels (332 tensors: 125 us of host time
// against 25).
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/scao_train.h"

namespace {

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SCAO_F32;
    case at::kBFloat16: return SCAO_BF16;
    case at::kHalf: return SCAO_F16;
    default: return -1;
  }
}

// gradients(parameters) -> (device index, count, table) or None.
// The gradients of a list or tuple of tensors, those that have one, as an array
// of scao_tensor_desc in a bytes object; None where any of them is not a dense
// fp32, bf16 or fp16 tensor on the first one's GPU whose elements fill their
// memory (in any order): those are for the caller to refuse or to copy.
PyObject* gradients(PyObject*, PyObject* arg) {
  PyObject* seq = PySequence_Fast(arg, "gradients() takes a list or a tuple");
  if (!seq) return nullptr;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject* out = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(scao_tensor_desc));
  if (!out) {
    Py_DECREF(seq);
    return nullptr;
  }
  auto* t = reinterpret_cast<scao_tensor_desc*>(PyBytes_AS_STRING(out));
  Py_ssize_t count = 0;
  int device = -1;
  bool plain = true;
  try {
    for (Py_ssize_t i = 0; i < n && plain; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
      if (!THPVariable_Check(o)) {
        plain = false;
        break;
      }
      const at::Tensor& g = THPVariable_Unpack(o).grad();
      if (!g.defined()) continue;
      const int code = g.layout() == at::kStrided && g.is_cuda() ? code_of(g.scalar_type()) : -1;
      plain = code >= 0 && (device < 0 || g.device().index() == device) &&
              g.is_non_overlapping_and_dense();
      if (!plain) break;
      device = g.device().index();
      t[count++] = scao_tensor_desc{g.data_ptr(), g.numel(), code, 0};
    }
  } catch (const std::exception&) {
    plain = false;   // the caller's way through Python says what is wrong
  }
  Py_DECREF(seq);
  if (!plain) {
    Py_DECREF(out);
    Py_RETURN_NONE;
  }
  return Py_BuildValue("inN", device, count, out);
}

PyMethodDef methods[] = {{"gradients", gradients, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
