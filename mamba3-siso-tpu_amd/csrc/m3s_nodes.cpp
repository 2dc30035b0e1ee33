// The embedding lookup as an autograd node in C++, over the C ABI's m3s_embed_fwd / m3s_embed_bwd.
//
// The lookup and its gradient are a launch or a few of 2 to 20 us at small batches, so the host decides
// what a call costs. torch's engine runs a node on a thread of its own; a node in Python then waits for
// the interpreter there, whose objects lie in another core's cache. Forward and backward of 64 tokens,
// D 768, took 80 us with a node in Python and take 42 with this one (torch's own embedding: 50); the
// lookup alone, without a gradient, 7.5 and 4.7. What is left is the engine's hand-over to its thread
// and back.
//
// The operators in 8 bits (eightbit.py) are here for the same reason, without a gradient: rows of a token
// take the device 2 to 6 us and took the host 8 to 12 in Python (a product of 256 float rows, two
// launches, 17).
//
// This module holds no mathematics and no launch of its own: the package's binding (_lib.py) hands it
// the loaded library's entry points. Each function takes dense tensors of the kernels' types and answers
// None for everything else, which the package then handles, or refuses, in Python.
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
  decltype(&m3s_rows8) rows8;   // by bind8()
  decltype(&m3s_rows8_values) values8;
  decltype(&m3s_matmul8) matmul8;
  decltype(&m3s_matmul8_takes_floats) takes_floats;
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

// ---- 8 bits -------------------------------------------------------------------------------------

constexpr int64_t kNormMax8 = 16384;   // the widest row that m3s_rows8 normalises

int64_t padded(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

bool float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
int32_t code(at::ScalarType t) { return t == at::kBFloat16 ? M3S_DTYPE_BF16 : M3S_DTYPE_F32; }

// A tensor that the argument is, or null: plain, on `device` if that is given, and without a gradient to take.
const Tensor* given(PyObject* o, const at::Device* device) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !plain(t) || (device && t.device() != *device) ||
      (at::GradMode::is_enabled() && t.requires_grad()))
    return nullptr;
  return &t;
}

// Rows of `t` (..., width) that run as one matrix of unit column stride: their count and stride.
bool row_matrix(const Tensor& t, int64_t& rows, int64_t& stride) {
  if (t.dim() < 1) return false;
  const int64_t width = t.size(-1);
  if (width < 1 || width > M3S_ROWS8_WIDTH_MAX) return false;
  rows = t.numel() / width;
  stride = width;
  if (rows < 1 || rows > M3S_ROWS8_MAX) return false;
  if (t.is_contiguous()) return true;
  if (t.dim() != 2 || (width > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < width)) return false;
  if (rows > 1) stride = t.stride(0);
  return true;
}

struct Rows {   // rows in 8 bits
  Tensor values, scales;
  int64_t rows = 0, width = 0;
};

Rows fresh_rows(int64_t rows, int64_t width, at::Device device, bool poison) {
  const int64_t steps = padded(width, 128) / 128;
  return {fresh({padded(rows, 16) / 16, steps, 2, 64, 16}, at::kFloat8_e4m3fn, device, poison),
          fresh({4 * steps, padded(rows, 128)}, at::kFloat8_e8m0fnu, device, poison), rows, width};
}

m3s_rows8_args rows8_args(const Tensor& x, int64_t stride, const Rows& out) {
  m3s_rows8_args a = {};
  a.struct_size = sizeof(a);
  a.x_dtype = code(x.scalar_type());
  a.width = (int32_t)out.width;
  a.rows = out.rows;
  a.x = x.data_ptr();
  a.ldx = stride;
  a.values = out.values.data_ptr();
  a.scales = out.scales.data_ptr();
  return a;
}

// The fields of a Rows8 (values, scales, width, lead) with the leading sizes of `shape`.
PyObject* wrap_rows(Rows& r, at::IntArrayRef lead) {
  PyObject* sizes = PyTuple_New((Py_ssize_t)lead.size());
  if (!sizes) return nullptr;
  for (size_t i = 0; i < lead.size(); ++i) PyTuple_SET_ITEM(sizes, i, PyLong_FromLongLong(lead[i]));
  return Py_BuildValue("(NNLN)", THPVariable_Wrap(std::move(r.values)), THPVariable_Wrap(std::move(r.scales)),
                       (long long)r.width, sizes);
}

// An int's value, -1 past 64 bits (Python refuses it).
int64_t whole_number(PyObject* o) {
  const int64_t n = PyLong_AsLongLong(o);
  if (n == -1) PyErr_Clear();
  return n;
}

// A Rows8 as the argument holds it.
bool unwrap_rows(PyObject* o, Rows& r, at::DimVector& lead) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
  const Tensor* values = given(PyTuple_GET_ITEM(o, 0), nullptr);
  if (!values) return false;
  const at::Device device = values->device();
  const Tensor* scales = given(PyTuple_GET_ITEM(o, 1), &device);
  PyObject *width = PyTuple_GET_ITEM(o, 2), *sizes = PyTuple_GET_ITEM(o, 3);
  if (!scales || !PyLong_Check(width) || !PyTuple_Check(sizes)) return false;
  r.width = whole_number(width);
  r.rows = 1;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(sizes); ++i) {
    PyObject* n = PyTuple_GET_ITEM(sizes, i);
    if (!PyLong_Check(n)) return false;
    const int64_t size = whole_number(n);
    if (size < 1 || size > M3S_ROWS8_MAX) return false;   // no rows: Python's
    lead.push_back(size);
    r.rows *= size;
    if (r.rows > M3S_ROWS8_MAX) return false;
  }
  if (r.width < 1 || r.width > M3S_ROWS8_WIDTH_MAX) return false;
  const int64_t steps = padded(r.width, 128) / 128;
  if (values->scalar_type() != at::kFloat8_e4m3fn || scales->scalar_type() != at::kFloat8_e8m0fnu ||
      values->sizes() != at::IntArrayRef({padded(r.rows, 16) / 16, steps, 2, 64, 16}) ||
      scales->sizes() != at::IntArrayRef({4 * steps, padded(r.rows, 128)}) || !values->is_contiguous() ||
      !scales->is_contiguous())
    return false;
  r.values = *values;
  r.scales = *scales;
  return true;
}

// rows8(x, gain or None, eps, add or None, poison): ((values, scales, width, lead), sum or None), or None.
PyObject* rows8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "rows8 takes rows, a gain, an epsilon, rows to add and a truth value");
    return nullptr;
  }
  TORCH_CHECK(lib.rows8, "rows8: the library's entry points are not bound");
  const double eps = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor* x = given(args[0], nullptr);
  int64_t rows = 0, stride = 0, add_rows = 0, add_stride = 0;
  if (!x || torch::jit::tracer::isTracing() || !float_type(x->scalar_type()) || !row_matrix(*x, rows, stride))
    Py_RETURN_NONE;
  const at::Device device = x->device();
  const int64_t width = x->size(-1);
  const Tensor *gain = nullptr, *add = nullptr;
  if (args[1] != Py_None) {
    gain = given(args[1], &device);
    if (!gain || gain->scalar_type() != at::kFloat || gain->dim() != 1 || gain->size(0) != width ||
        !gain->is_contiguous() || width > kNormMax8 || reinterpret_cast<uintptr_t>(gain->data_ptr()) % 16)
      Py_RETURN_NONE;
  }
  if (args[3] != Py_None) {
    add = given(args[3], &device);
    if (!add || !gain || add->scalar_type() != at::kBFloat16 || add->sizes() != x->sizes() ||
        !row_matrix(*add, add_rows, add_stride))
      Py_RETURN_NONE;
  }
  const c10::DeviceGuard guard(device);
  const bool poison = args[4] == Py_True;
  Rows out = fresh_rows(rows, width, device, poison);
  m3s_rows8_args a = rows8_args(*x, stride, out);
  a.eps = (float)eps;
  Tensor sum;
  if (gain) a.gain = static_cast<const float*>(gain->data_ptr());
  if (add) {
    sum = fresh(x->sizes(), x->scalar_type(), device, poison);
    a.add = add->data_ptr();
    a.ldadd = add_stride;
    a.sum = sum.data_ptr();
  }
  check(lib.rows8(&a, stream_of(device)), "m3s_rows8");
  PyObject* r = wrap_rows(out, x->sizes().slice(0, x->dim() - 1));
  if (!r) return nullptr;
  if (add) return Py_BuildValue("(NN)", r, THPVariable_Wrap(std::move(sum)));
  return Py_BuildValue("(NO)", r, Py_None);
  END_HANDLE_TH_ERRORS
}

// rows8_values(rows, bf16 (else float32), poison): the values that a Rows8 stands for, or None.
PyObject* rows8_values(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3) {
    PyErr_SetString(PyExc_TypeError, "rows8_values takes rows and two truth values");
    return nullptr;
  }
  TORCH_CHECK(lib.values8, "rows8_values: the library's entry points are not bound");
  Rows r;
  at::DimVector sizes;
  if (torch::jit::tracer::isTracing() || !unwrap_rows(args[0], r, sizes)) Py_RETURN_NONE;
  const at::Device device = r.values.device();
  const c10::DeviceGuard guard(device);
  sizes.push_back(r.width);
  const at::ScalarType type = args[1] == Py_True ? at::kBFloat16 : at::kFloat;
  Tensor y = fresh(sizes, type, device, args[2] == Py_True);
  m3s_rows8_values_args a = {};
  a.struct_size = sizeof(a);
  a.y_dtype = code(type);
  a.width = (int32_t)r.width;
  a.rows = r.rows;
  a.values = r.values.data_ptr();
  a.scales = r.scales.data_ptr();
  a.y = y.data_ptr();
  check(lib.values8(&a, stream_of(device)), "m3s_rows8_values");
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// matmul8(rows, weight, gated, activation, bias or None, residual or None, poison): the product, gated a
// Rows8's fields, or None. `rows` is a tensor or a Rows8, `weight` a Weight8.
PyObject* matmul8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7) {
    PyErr_SetString(PyExc_TypeError,
                    "matmul8 takes rows, a weight, a truth value, an activation, a bias, a residual and a truth value");
    return nullptr;
  }
  TORCH_CHECK(lib.matmul8 && lib.rows8, "matmul8: the library's entry points are not bound");
  const int64_t activation = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  PyObject* wt = args[1];
  const bool gated = args[2] == Py_True;
  if (torch::jit::tracer::isTracing() || !PyTuple_Check(wt) || PyTuple_GET_SIZE(wt) != 6 ||
      PyTuple_GET_ITEM(wt, 4) != (gated ? Py_True : Py_False) || !PyBool_Check(PyTuple_GET_ITEM(wt, 5)) ||
      !PyLong_Check(PyTuple_GET_ITEM(wt, 2)) ||
      !PyLong_Check(PyTuple_GET_ITEM(wt, 3)))
    Py_RETURN_NONE;
  const Tensor* wv = given(PyTuple_GET_ITEM(wt, 0), nullptr);
  if (!wv) Py_RETURN_NONE;
  const at::Device device = wv->device();
  const Tensor* wsc = given(PyTuple_GET_ITEM(wt, 1), &device);
  const int64_t k = whole_number(PyTuple_GET_ITEM(wt, 2)), n = whole_number(PyTuple_GET_ITEM(wt, 3));
  if (!wsc || k < 1 || k > M3S_ROWS8_WIDTH_MAX || n < 1 || n > M3S_ROWS8_WIDTH_MAX) Py_RETURN_NONE;
  const int64_t tiles = (gated ? 2 * padded(n, 128) : padded(n, 64)) / 16, steps = padded(k, 128) / 128;
  if (wv->sizes() != at::IntArrayRef({tiles, steps, 2, 64, 16}) || wv->scalar_type() != at::kFloat8_e4m3fn ||
      wsc->sizes() != at::IntArrayRef({steps, tiles / 4, 64, 4}) || wsc->scalar_type() != at::kFloat8_e8m0fnu ||
      !wv->is_contiguous() || !wsc->is_contiguous())
    Py_RETURN_NONE;
  m3s_matmul8_args a = {};
  a.struct_size = sizeof(a);
  a.k = (int32_t)k;
  a.n = (int32_t)n;
  a.gated = gated;
  a.activation = (int32_t)activation;
  a.short_sums = PyTuple_GET_ITEM(wt, 5) == Py_True;
  a.w = wv->data_ptr();
  a.w_scales = wsc->data_ptr();
  Rows r;
  at::DimVector lead;
  const Tensor* x = nullptr;
  int64_t stride = 0;
  if (THPVariable_Check(args[0])) {
    x = given(args[0], &device);
    if (!x || !float_type(x->scalar_type()) || !row_matrix(*x, r.rows, stride)) Py_RETURN_NONE;
    r.width = x->size(-1);
    lead.append(x->sizes().begin(), x->sizes().end() - 1);
  } else if (!unwrap_rows(args[0], r, lead) || r.values.device() != device) {
    Py_RETURN_NONE;
  }
  if (r.width != k) Py_RETURN_NONE;
  at::DimVector sizes = lead;
  sizes.push_back(n);
  if (args[4] != Py_None) {
    const Tensor* bias = given(args[4], &device);
    if (!bias || bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != (gated ? 2 * n : n) ||
        !bias->is_contiguous())
      Py_RETURN_NONE;
    a.bias = static_cast<const float*>(bias->data_ptr());
  }
  if (args[5] != Py_None) {
    const Tensor* res = given(args[5], &device);
    int64_t rows = 0;
    if (!res || gated || res->scalar_type() != at::kBFloat16 || res->sizes() != at::IntArrayRef(sizes) ||
        !row_matrix(*res, rows, a.ldres))
      Py_RETURN_NONE;
    a.residual = res->data_ptr();
  }
  const c10::DeviceGuard guard(device);
  const bool poison = args[6] == Py_True;
  void* stream = stream_of(device);
  if (x && !lib.takes_floats(r.rows, a.k, a.n, gated, code(x->scalar_type()))) {
    r = fresh_rows(r.rows, r.width, device, poison);
    m3s_rows8_args q = rows8_args(*x, stride, r);
    check(lib.rows8(&q, stream), "m3s_rows8");
    x = nullptr;
  }
  a.rows = r.rows;
  if (x) {
    a.x_dtype = code(x->scalar_type());
    a.x = x->data_ptr();
    a.ldx = stride;
  } else {
    a.x_dtype = M3S_DTYPE_ROWS8;
    a.x = r.values.data_ptr();
    a.x_scales = r.scales.data_ptr();
  }
  if (gated) {
    Rows out = fresh_rows(r.rows, n, device, poison);
    a.y_values = out.values.data_ptr();
    a.y_scales = out.scales.data_ptr();
    check(lib.matmul8(&a, stream), "m3s_matmul8");
    return wrap_rows(out, lead);
  }
  Tensor y = fresh(sizes, at::kBFloat16, device, poison);
  a.y = y.data_ptr();
  a.ldy = n;
  check(lib.matmul8(&a, stream), "m3s_matmul8");
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

bool addresses(PyObject* const* args, Py_ssize_t nargs, void** at, Py_ssize_t count) {
  if (nargs != count) {
    PyErr_Format(PyExc_TypeError, "takes %zd addresses", count);
    return false;
  }
  for (Py_ssize_t i = 0; i < count; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return false;
  }
  return true;
}

// bind8(m3s_rows8, m3s_rows8_values, m3s_matmul8, m3s_matmul8_takes_floats): addresses.
PyObject* bind8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* at[4];
  if (!addresses(args, nargs, at, 4)) return nullptr;
  lib.rows8 = reinterpret_cast<decltype(lib.rows8)>(at[0]);
  lib.values8 = reinterpret_cast<decltype(lib.values8)>(at[1]);
  lib.matmul8 = reinterpret_cast<decltype(lib.matmul8)>(at[2]);
  lib.takes_floats = reinterpret_cast<decltype(lib.takes_floats)>(at[3]);
  Py_RETURN_NONE;
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
    {"rows8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows8)), METH_FASTCALL, nullptr},
    {"rows8_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows8_values)), METH_FASTCALL, nullptr},
    {"matmul8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(matmul8)), METH_FASTCALL, nullptr},
    {"bind8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind8)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "m3s_nodes", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_m3s_nodes(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) return nullptr;
  return m;
}
