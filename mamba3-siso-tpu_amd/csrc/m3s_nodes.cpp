// The embedding lookup as an autograd node in C++, over the C ABI's m3s_embed_fwd / m3s_embed_bwd.
//
// The lookup and its gradient are a launch or a few of 2 to 20 us at small batches, so the host decides
// what a call costs. torch's engine runs a node on a thread of its own; a node in Python then waits for
// the interpreter there, whose objects lie in another core's cache. Forward and backward of 64 tokens,
// D 768, took 80 us with a node in Python and take 42 with this one (torch's own embedding: 50); the
// lookup alone, without a gradient, 7.5 and 4.7. What is left is the engine's hand-over to its thread
// and back.
//
// This module holds no mathematics and no launch of its own: the package's binding (_lib.py) hands it
// the loaded library's entry points. embed() takes dense tensors of the kernels' types and answers None
// for everything else, which the package then handles, or refuses, in Python.
#include <Python.h>

#include <mutex>
#include <string>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/version.h>

#include "../../include/m3s.h"

namespace {

using at::Tensor;
namespace ag = torch::autograd;

struct Entries {   // of the loaded library, by bind()
  decltype(&m3s_embed_fwd) fwd;
  decltype(&m3s_embed_bwd) bwd;
  decltype(&m3s_embed_bwd_workspace_bytes) bwd_bytes;
  decltype(&m3s_last_error) error;
} lib = {};

// The exception types of the Python binding's check().
void check(int32_t rc, const char* who) {
  if (rc == M3S_OK) return;
  const std::string msg = std::string(who) + ": " + lib.error();
  TORCH_CHECK_VALUE(rc != M3S_ERR_INVALID && rc != M3S_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, msg);
}

// An output or workspace; `poison` fills it with ones (NaN in every float type), as the package does
// where tests look for memory that a kernel leaves unwritten.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, at::Device device, bool poison) {
  Tensor t = at::empty(sizes, at::TensorOptions().dtype(type).device(device));
  if (poison && t.numel()) t.view(-1).view(at::kByte).fill_(255);
  return t;
}

m3s_embed_args embed_args(const Tensor& tokens, at::ScalarType type, int64_t vocab, int64_t width, float scale,
                          int64_t pad) {
  m3s_embed_args a = {};
  a.struct_size = sizeof(a);
  a.dtype = type == at::kBFloat16 ? M3S_DTYPE_BF16 : M3S_DTYPE_F32;
  a.id_bytes = (int32_t)tokens.element_size();
  a.vocab = (int32_t)vocab;
  a.width = (int32_t)width;
  a.scale = scale;
  a.tokens = tokens.numel();
  a.padding_idx = pad;
  a.ids = tokens.data_ptr();
  return a;
}

void* stream_of(at::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

bool ids_type(at::ScalarType t) { return t == at::kLong || t == at::kInt; }

// The gradient of the table; differentiable once.
struct EmbedBackward : public ag::Node {
  ag::SavedVariable tokens_;
  int64_t vocab = 0, width = 0, pad = -1;
  float scale = 1.f;
  at::ScalarType type = at::kFloat;
  bool poison = false;

  std::string name() const override { return "M3sEmbedBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens_.reset_data();
  }

  ag::variable_list apply(ag::variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const Tensor given = grads[0].defined() ? grads[0] : input_metadata(0).zeros_like();
    const Tensor saved = tokens_.unpack();
    Tensor dtable;
    {
      at::AutoGradMode no_graph(false);
      const at::Device device = given.device();
      // what hooks on saved tensors brought back may lie anywhere
      TORCH_CHECK_VALUE(saved.device() == device && ids_type(saved.scalar_type()) && given.scalar_type() == type &&
                            given.numel() == saved.numel() * width,
                        "embedding: the saved tokens came back as another kind of tensor");
      const c10::DeviceGuard guard(device);
      const Tensor tokens = saved.contiguous(), dy = given.contiguous();
      m3s_embed_args a = embed_args(tokens, type, vocab, width, scale, pad);
      const int64_t nbytes = lib.bwd_bytes(a.tokens, a.vocab, a.width);
      TORCH_CHECK_VALUE(nbytes >= 0, "embedding: bad sizes (tokens ", a.tokens, ", vocab ", vocab, ", width ", width,
                        ")");
      dtable = fresh({vocab, width}, type, device, poison);
      Tensor workspace;
      if (nbytes) {
        workspace = fresh({nbytes}, at::kByte, device, poison);
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = nbytes;
      }
      a.dy = dy.data_ptr();
      a.dtable = dtable.data_ptr();
      check(lib.bwd(&a, stream_of(device)), "m3s_embed_bwd");
    }
    if (at::GradMode::is_enabled() && given.requires_grad()) {   // no second derivative: say so when it is asked for
      ag::set_history(dtable, std::shared_ptr<ag::Error>(
                                  new ag::Error("trying to differentiate twice a function that is differentiable once",
                                                ag::collect_next_edges(given)),
                                  ag::deleteNode));
    }
    return {dtable};
  }
};

// A strided tensor on a GPU that is nothing but its values: no subclass, no transform's wrapper, and no
// tangent.
bool plain(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && !at::isTensorSubclassLike(t) && !t.is_neg() &&
         !t._fw_grad(0).defined();
}

bool takes(const Tensor& table, const Tensor& tokens) {
  if (!table.defined() || !tokens.defined() || torch::jit::tracer::isTracing()) return false;
  if (!plain(table) || !plain(tokens) || tokens.device() != table.device() || table.dim() != 2) return false;
  const int64_t v = table.size(0), d = table.size(1);
  const auto type = table.scalar_type();
  return v > 0 && v < INT32_MAX && d > 0 && d < 1 << 22 && tokens.numel() < INT32_MAX - 63 &&
         (table.stride(1) == 1 || d == 1) && (type == at::kFloat || type == at::kBFloat16) &&
         ids_type(tokens.scalar_type()) && tokens.is_contiguous();
}

// embed(table, tokens, scale, padding id or -1, poison): the looked up rows, or None.
PyObject* embed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "embed takes a table, tokens, a scale, a padding id and a truth value");
    return nullptr;
  }
  TORCH_CHECK(lib.fwd, "embed: the library's entry points are not bound");
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) Py_RETURN_NONE;
  const Tensor& table = THPVariable_Unpack(args[0]);
  const Tensor& tokens = THPVariable_Unpack(args[1]);
  const double scale = PyFloat_AsDouble(args[2]);
  const int64_t pad = PyLong_AsLongLong(args[3]);
  const bool poison = args[4] == Py_True;
  if (PyErr_Occurred()) return nullptr;
  if (!takes(table, tokens)) Py_RETURN_NONE;

  const c10::DeviceGuard guard(table.device());
  at::DimVector sizes(tokens.sizes().begin(), tokens.sizes().end());
  sizes.push_back(table.size(1));
  Tensor y = fresh(sizes, table.scalar_type(), table.device(), poison);
  m3s_embed_args a = embed_args(tokens, table.scalar_type(), table.size(0), table.size(1), (float)scale, pad);
  a.table = table.data_ptr();
  a.table_stride = table.stride(0);
  a.y = y.data_ptr();
  check(lib.fwd(&a, stream_of(table.device())), "m3s_embed_fwd");
  if (at::GradMode::is_enabled() && table.requires_grad()) {
    std::shared_ptr<EmbedBackward> node(new EmbedBackward(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(table));
    node->tokens_ = ag::SavedVariable(tokens, false);
    node->vocab = table.size(0);
    node->width = table.size(1);
    node->pad = pad;
    node->scale = (float)scale;
    node->type = table.scalar_type();
    node->poison = poison;
    ag::set_history(y, node);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// bind(m3s_embed_fwd, m3s_embed_bwd, m3s_embed_bwd_workspace_bytes, m3s_last_error): addresses.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* at[4];
  if (nargs != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
    return nullptr;
  }
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib.fwd = reinterpret_cast<decltype(lib.fwd)>(at[0]);
  lib.bwd = reinterpret_cast<decltype(lib.bwd)>(at[1]);
  lib.bwd_bytes = reinterpret_cast<decltype(lib.bwd_bytes)>(at[2]);
  lib.error = reinterpret_cast<decltype(lib.error)>(at[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"embed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(embed)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "m3s_nodes", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_m3s_nodes(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) return nullptr;
  return m;
}
