// The embedding's autograd node. As a node in Python a training pass of few tokens takes
// twice as long: autograd runs the backward on a thread of its own, so what Python
// touches (the interpreter, its objects, the allocator's and the stream's state) moves
// from core to core and back in every pass. 200 ids into 300 x 64, lookup and gradient:
// 80 to 86 us by host as model_ops._EmbeddingFn, 47 here (torch's nn.Embedding 50; the
// hand-over to the other thread and back alone some 35).
//
// The same function as model_ops._EmbeddingFn for bf16 and fp32 tables and outputs. What
// its gradient's kernels do not take (a graph of the gradient, batched gradients) is
// Python's as there.
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/ngdn.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// model_ops' gradient and _lib.NgdnError, for the life of the process
py::object *python_grad = nullptr, *ngdn_error = nullptr;

struct Failed : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void done(int32_t rc, const char* what) {
  if (rc) throw Failed(std::string(what) + " failed (" + std::to_string(rc) + "): " + ngdn_last_error());
}

int32_t code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? NGDN_BF16 : NGDN_F32; }

void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding,
                        at::ScalarType type) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["type"] = (int64_t)weight.scalar_type();
    const c10::DeviceGuard guard(weight.device());
    const Tensor w = weight.contiguous();
    std::vector<int64_t> shape = ids.sizes().vec();
    shape.push_back(w.size(1));
    Tensor y = at::empty(shape, w.options().dtype(type));
    if (ids.numel() > 0)
      done(ngdn_embedding_fwd(code(w), code(y), ids.numel(), w.size(0), (int32_t)w.size(1), (float)scale,
                              ids.const_data_ptr<int64_t>(), w.const_data_ptr(), y.mutable_data_ptr(), stream(w)),
           "ngdn_embedding_fwd");
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t padding = ctx->saved_data["padding"].toInt(), V = ctx->saved_data["rows"].toInt();
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const Tensor& g = grads[0];
    if (at::GradMode::is_enabled() || !g.has_storage() || g.key_set().has(c10::DispatchKey::Python)) {
      const py::gil_scoped_acquire gil;
      const py::object pad = padding < 0 ? py::object(py::none()) : py::cast(padding);
      return {Tensor(), (*python_grad)(ids, g, scale, pad, V, type).cast<Tensor>(), Tensor(), Tensor(), Tensor()};
    }
    const c10::DeviceGuard guard(g.device());
    const Tensor dy = g.contiguous();
    const int64_t N = ids.numel(), D = dy.size(-1);
    Tensor dw = at::empty({V, D}, dy.options().dtype(type));
    const Tensor ws = at::empty({(ngdn_embedding_ws(N, V, (int32_t)D) + 1) / 2}, ids.options());
    done(ngdn_embedding_bwd(code(dy), code(dw), N, V, (int32_t)D, (float)scale, padding, ids.const_data_ptr<int64_t>(),
                            dy.const_data_ptr(), dw.mutable_data_ptr(), static_cast<int32_t*>(ws.mutable_data_ptr()),
                            stream(dy)),
         "ngdn_embedding_bwd");
    return {Tensor(), dw, Tensor(), Tensor(), Tensor()};
  }
};

// ids int64 and contiguous, weight [V,D] on the same GPU, both types as above
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, int64_t padding, at::ScalarType type) {
  try {
    const py::gil_scoped_release off;
    return EmbeddingFn::apply(ids, weight, scale, padding, type);
  } catch (const Failed& e) {
    PyErr_SetString(ngdn_error->ptr(), e.what());
    throw py::error_already_set();
  }
}

}  // namespace

PYBIND11_MODULE(_node, m) {
  // a tensor's grad_fn in Python, by the name that the function has there
  static PyTypeObject grad_fn;
  torch::autograd::_initFunctionPyTypeObject(grad_fn, "_EmbeddingFnBackward", nullptr, nullptr);
  torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<EmbeddingFn>), &grad_fn);
  m.attr("version") = NGDN_VERSION;
  m.def("setup", [](py::object grad, py::object error) {
    python_grad = new py::object(std::move(grad));
    ngdn_error = new py::object(std::move(error));
  });
  m.def("embedding", &embedding);
}
