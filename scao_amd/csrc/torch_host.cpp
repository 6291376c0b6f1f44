// The Python module scao_amd._torch_host: what would cost more host time in
// Python than the kernels take.
//
//   gradients   the table of a model's gradients (scao_tensor_desc): reading six
//               properties of 332 tensors from Python takes 125 us, their norm
//               and scaling 25
//   gated_ffn   the feed-forward block as a node of torch's graph, its backward
//               pass without the interpreter: a small block's training step took
//               145 us of host time as a Python function
//   bind        the addresses of the C ABI's entry points, which the caller has
//               loaded (so that one library is used, whichever it is)
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/scao_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&scao_last_error) last_error;
  decltype(&scao_ffn_saved_bytes) saved_bytes;
  decltype(&scao_ffn_forward_workspace) forward_workspace;
  decltype(&scao_ffn_forward) forward;
  decltype(&scao_ffn_backward_workspace) backward_workspace;
  decltype(&scao_ffn_backward) backward;
} lib;

void check(int rc, const char* who) {
  TORCH_CHECK(rc == SCAO_OK, who, " failed (", rc, "): ", lib.last_error());
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SCAO_F32;
    case at::kBFloat16: return SCAO_BF16;
    case at::kHalf: return SCAO_F16;
    default: return -1;
  }
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({n}, like.options().dtype(at::kByte));
}

// ------------------------------------------------------------- gated_ffn ---
constexpr int64_t MAX_STRIDE = (int64_t)1 << 21;   // of rows that scao_ffn_* take

// x, w_gate, w_up, w_down: 2-D, unit column stride, rows that do not overlap,
// matching sizes, type and device (the caller has checked them)
scao_ffn_desc describe(const Tensor& x, const Tensor& g, const Tensor& u, const Tensor& d,
                       int64_t act) {
  return scao_ffn_desc{x.data_ptr(),  g.data_ptr(),  u.data_ptr(),        d.data_ptr(),
                       x.stride(0),   g.stride(0),   u.stride(0),         d.stride(0),
                       x.size(0),     g.size(1),     g.size(0),           code_of(x.scalar_type()),
                       (int32_t)act};
}

std::pair<Tensor, Tensor> forward(const Tensor& x, const Tensor& g, const Tensor& u,
                                  const Tensor& d, int64_t act, bool save) {
  const c10::DeviceGuard guard(x.device());
  const scao_ffn_desc desc = describe(x, g, u, d, act);
  Tensor y = at::empty({x.size(0), x.size(1)}, x.options().requires_grad(false)), saved;
  if (save) saved = bytes(lib.saved_bytes(&desc), x);
  const Tensor work = bytes(lib.forward_workspace(&desc, save), x);
  check(lib.forward(&desc, y.data_ptr(), save ? saved.data_ptr() : nullptr, work.data_ptr(),
                    stream_of(x)),
        "scao_ffn_forward");
  return {y, saved};
}

struct GatedFFN : torch::autograd::Function<GatedFFN> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const Tensor& u,
                        const Tensor& d, int64_t act) {
    auto [y, saved] = ::forward(x, g, u, d, act, true);
    ctx->save_for_backward({x, g, u, d, saved});
    ctx->saved_data["act"] = act;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (hooks on saved tensors may have moved them: their addresses are new)
    const variable_list t = ctx->get_saved_variables();
    const Tensor &x = t[0], &g = t[1], &u = t[2], &d = t[3], &saved = t[4];
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const bool higher = at::GradMode::is_enabled();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      Tensor dy = grads[0];
      if ((dy.stride(1) != 1 && dy.size(1) != 1) ||
          (dy.size(0) > 1 && (dy.stride(0) < dy.size(1) || dy.stride(0) >= MAX_STRIDE)))
        dy = dy.contiguous();
      const scao_ffn_desc desc = describe(x, g, u, d, ctx->saved_data["act"].toInt());
      int want = 0;
      const Tensor* like[4] = {&x, &g, &u, &d};
      void* to[4] = {};
      for (int i = 0; i < 4; ++i) {
        if (!ctx->needs_input_grad(i)) continue;
        want |= 1 << i;
        out[i] = at::empty({like[i]->size(0), like[i]->size(1)},
                           x.options().requires_grad(false));
        to[i] = out[i].data_ptr();
      }
      static_assert(SCAO_FFN_DX == 1 && SCAO_FFN_DGATE == 2 && SCAO_FFN_DUP == 4 &&
                        SCAO_FFN_DDOWN == 8,
                    "the inputs' order");
      const Tensor work =
          bytes(lib.backward_workspace(&desc, dy.data_ptr(), dy.stride(0), want), x);
      check(lib.backward(&desc, dy.data_ptr(), dy.stride(0), saved.data_ptr(), to[0], to[1], to[2],
                         to[3], work.data_ptr(), stream_of(x)),
            "scao_ffn_backward");
    }
    if (higher) {   // a gradient of these gradients is an error, not a zero
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "gated_ffn is differentiable once", 4);
      variable_list have;
      for (int i = 0; i < 4; ++i)
        if (out[i].defined()) have.push_back(out[i].requires_grad_(true));
      have = (*error)(std::move(have));
      for (int i = 0, k = 0; i < 4; ++i)
        if (out[i].defined()) out[i] = have[k++];
    }
    return out;
  }
};

PyObject* gated_ffn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "gated_ffn() takes five arguments");
  for (int i = 0; i < 4; ++i)
    TORCH_CHECK_TYPE(THPVariable_Check(args[i]), "gated_ffn() takes tensors");
  const long act = PyLong_AsLong(args[4]);
  if (act == -1 && PyErr_Occurred()) return nullptr;
  const Tensor &x = THPVariable_Unpack(args[0]), &g = THPVariable_Unpack(args[1]),
               &u = THPVariable_Unpack(args[2]), &d = THPVariable_Unpack(args[3]);
  for (const Tensor* t : {&x, &g, &u, &d})
    TORCH_CHECK(t->dim() == 2 && (t->stride(1) == 1 || t->size(1) == 1), "gated_ffn() takes rows");
  if (at::GradMode::is_enabled() && (x.requires_grad() || g.requires_grad() ||
                                     u.requires_grad() || d.requires_grad()))
    return THPVariable_Wrap(GatedFFN::apply(x, g, u, d, (int64_t)act));
  return THPVariable_Wrap(forward(x, g, u, d, act, false).first);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------- gradients ---
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
      const Tensor& g = THPVariable_Unpack(o).grad();
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

// bind({name: address})
PyObject* bind(PyObject*, PyObject* arg) {
  auto at = [&](const char* name, auto& entry) {
    PyObject* v = PyDict_Check(arg) ? PyDict_GetItemString(arg, name) : nullptr;
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!p && !PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "bind() has no %s", name);
    entry = reinterpret_cast<std::decay_t<decltype(entry)>>(p);
    return p != nullptr;
  };
  if (!(at("scao_last_error", lib.last_error) && at("scao_ffn_saved_bytes", lib.saved_bytes) &&
        at("scao_ffn_forward_workspace", lib.forward_workspace) &&
        at("scao_ffn_forward", lib.forward) &&
        at("scao_ffn_backward_workspace", lib.backward_workspace) &&
        at("scao_ffn_backward", lib.backward)))
    return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"gradients", gradients, METH_O, nullptr},
    {"gated_ffn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gated_ffn)),
     METH_FASTCALL, nullptr},
    {"bind", bind, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_host", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_host(void) { return PyModule_Create(&module); }
