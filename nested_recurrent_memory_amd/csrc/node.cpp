// Autograd nodes over the library: the embedding's, dropout's and the residual norm's,
// and the sampler's call. As a node in Python, the embedding's training pass of few tokens takes
// twice as long: autograd runs the backward on a thread of its own, so what Python
// touches (the interpreter, its objects, the allocator's and the stream's state) moves
// from core to core and back in every pass. 200 ids into 300 x 64, lookup and gradient:
// 80 to 86 us by host as model_ops._EmbeddingFn, 47 here (torch's nn.Embedding 50; the
// hand-over to the other thread and back alone some 35).
//
// The embedding is the same function as model_ops._EmbeddingFn for bf16 and fp32 tables and outputs. What
// its gradient's kernels do not take (a graph of the gradient, batched gradients) is
// Python's as there.
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_cpp_function.h>
#include <torch/csrc/autograd/python_variable.h>
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

// ---------------------------------------------------------------- dropout, the residual norm, the sampler

using Optional = c10::optional<Tensor>;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

void on_gpu(const char* name, const Tensor& t, const Tensor& first) {
  if (!t.is_cuda() || t.device() != first.device())
    refuse(std::string(name) + ": every tensor must be on one GPU (got " + t.device().str() + "); there is no CPU path");
}

bool floats(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf;
}

void check_floats(const char* name, const char* which, const Tensor& t) {
  if (!floats(t)) refuse(std::string(name) + ": " + which + " is " + c10::toString(t.scalar_type()) + " (bf16, fp16 or fp32)");
}

Tensor given(const Optional& t) { return t ? *t : Tensor(); }

// fp16 runs in fp32
Tensor widened(const Tensor& t) { return t.defined() && t.scalar_type() == at::kHalf ? t.to(at::kFloat) : t; }

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// outside a node nothing would carry a tangent on
void no_tangents(const char* name, std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    if (t.defined() && t._fw_grad(0).defined())
      throw std::runtime_error(std::string(name) + ": forward-mode differentiation is not supported");
}

// Where words come from: an integer (modulo 2^64) or one int64 on the GPU, and a number.
struct Stream {
  int64_t seed = 0, offset = 0, threshold = 0;
  Tensor seed_tensor;
  double p = 0;
  float keep() const { return p < 1 ? (float)(1 / (1 - p)) : 0.f; }
};

int64_t word(const py::object& v, const char* name, const char* which) {
  if (!PyIndex_Check(v.ptr()) || PyBool_Check(v.ptr()))
    refuse(std::string(name) + ": " + which + " must be an integer");
  const py::object i = py::reinterpret_steal<py::object>(PyNumber_Index(v.ptr()));
  if (!i) throw py::error_already_set();
  return (int64_t)PyLong_AsUnsignedLongLongMask(i.ptr());
}

Stream stream_from(const char* name, double p, const py::object& seed, const py::object& offset) {
  Stream s;
  if (!(p >= 0 && p <= 1)) refuse(std::string(name) + ": p " + std::to_string(p) + " outside [0, 1]");
  s.p = p;
  s.threshold = (int64_t)std::nearbyint(p * 4294967296.0);
  if (THPVariable_Check(seed.ptr())) {
    const Tensor t = THPVariable_Unpack(seed.ptr());
    if (t.scalar_type() != at::kLong || t.numel() != 1)
      refuse(std::string(name) + ": a seed tensor holds one int64, got " + c10::toString(t.scalar_type()) + " " + shape(t));
    s.seed_tensor = t;
  } else {
    s.seed = word(seed, name, "seed");
  }
  s.offset = word(offset, name, "offset");
  return s;
}

// t with its values in memory as they are read, row by row: contiguous, and not a view
// that stands for their negatives (an imaginary part of a conjugate)
Tensor whole(const Tensor& t) { return t.defined() ? t.contiguous().resolve_neg() : t; }

// A pointer for a kernel: of memory on the GPU, which tensors of function transforms, fake
// ones and other subclasses with a dispatch of their own do not hold. Null where undefined.
const void* raw(const Tensor& t) {
  if (!t.defined()) return nullptr;
  if (!t.has_storage() || t.key_set().has(c10::DispatchKey::Python))
    throw std::runtime_error("the library's kernels take plain tensors: function transforms, tracers and tensor "
                             "subclasses are not supported");
  if (t.numel() > 0) {
    // a parameter whose memory has been taken back for now (sharded training) still has its shape
    int64_t end = t.storage_offset() + 1;
    for (int64_t d = 0; d < t.dim(); ++d) end += (t.size(d) - 1) * t.stride(d);
    if ((size_t)end * t.element_size() > t.storage().nbytes())
      throw std::runtime_error("a tensor's memory does not hold it (released, or not yet there)");
  }
  return t.const_data_ptr();
}
void* raw_out(const Tensor& t) {
  return raw(t) ? t.mutable_data_ptr() : nullptr;
}

const int64_t* seed_of(const Tensor& t) { return static_cast<const int64_t*>(raw(t)); }

void plain_gradient(const char* name, const Tensor& g) {
  if (g.defined() && !g.has_storage())
    throw std::runtime_error(std::string(name) + ": gradients of several outputs at once (is_grads_batched, vmap) are not supported");
}

Tensor drop(const Tensor& x, const Stream& s) {
  const c10::DeviceGuard guard(x.device());
  const Tensor c = whole(x);
  Tensor y = at::empty_like(c);
  done(ngdn_dropout(code(c), c.numel(), s.threshold, s.keep(), s.seed, seed_of(s.seed_tensor), s.offset,
                    raw(c), raw_out(y), stream(c)),
       "ngdn_dropout");
  return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Stream& s) {
    if (s.seed_tensor.defined()) ctx->save_for_backward({s.seed_tensor});
    ctx->saved_data["seed"] = s.seed;
    ctx->saved_data["offset"] = s.offset;
    ctx->saved_data["threshold"] = s.threshold;
    ctx->saved_data["p"] = s.p;
    return drop(x, s);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Stream s;
    const auto saved = ctx->get_saved_variables();
    if (!saved.empty()) s.seed_tensor = saved[0];
    s.seed = ctx->saved_data["seed"].toInt();
    s.offset = ctx->saved_data["offset"].toInt();
    s.threshold = ctx->saved_data["threshold"].toInt();
    s.p = ctx->saved_data["p"].toDouble();
    plain_gradient("dropout", grads[0]);
    // linear in x: its gradient is dropout of the gradient, to any order
    if (at::GradMode::is_enabled()) return {DropoutFn::apply(grads[0], s), Tensor()};
    return {drop(grads[0], s), Tensor()};
  }
};

Tensor dropout(const Tensor& x, double p, const py::object& seed, const py::object& offset) {
  check_floats("dropout", "x", x);
  const Stream s = stream_from("dropout", p, seed, offset);
  on_gpu("dropout", x, x);
  if (s.seed_tensor.defined()) on_gpu("dropout", s.seed_tensor, x);
  if (s.threshold == 0) return x;
  const py::gil_scoped_release free;        // a launch may wait for room in the queue
  const Tensor w = widened(x);
  Tensor y;
  if (wants_grad({w})) {
    y = DropoutFn::apply(w, s);
  } else {
    no_tangents("dropout", {w});
    y = drop(w.detach(), s);
  }
  return y.scalar_type() == x.scalar_type() ? y : y.to(x.scalar_type());
}

// a residual norm's scalars, kept for its backward
struct Residual : torch::CustomClassHolder {
  ngdn_residual_args a{};
  at::ScalarType y_type = at::kFloat;
};

// its tensors: x, branch, weight, post_weight, gate and the seed, undefined where not given
using Parts = std::array<Tensor, 6>;

struct Seed {       // a tensor that autograd does not take for an input
  Tensor t;
};

void point(ngdn_residual_args& a, const Parts& t) {
  a.x = raw(t[0]); a.branch = raw(t[1]); a.weight = raw(t[2]); a.post_weight = raw(t[3]);
  a.gate = raw(t[4]); a.seed_ptr = seed_of(t[5]);
}

Parts whole(const Parts& t) {
  Parts c;
  for (int i = 0; i < 6; ++i) c[i] = whole(t[i]);
  return c;
}

// h, y (undefined without weight) and the two statistics (where saved is set)
void residual_forward(const Parts& t, const Residual& r, Tensor* out, bool saved) {
  ngdn_residual_args a = r.a;
  point(a, t);
  out[0] = at::empty_like(t[0]);
  a.h = raw_out(out[0]);
  if (t[2].defined()) {
    out[1] = at::empty_like(t[0], t[0].options().dtype(r.y_type));
    a.y = raw_out(out[1]);
  }
  if (saved) {
    out[2] = at::empty({2, a.rows}, t[0].options().dtype(at::kFloat));
    a.rstd_h = static_cast<float*>(raw_out(out[2]));
    a.rstd_b = a.rstd_h + a.rows;
  }
  done(ngdn_residual_norm_fwd(&a, stream(t[0])), "ngdn_residual_norm_fwd");
}

struct ResidualFn : torch::autograd::Function<ResidualFn> {
  // given: those of x, branch, weight, post_weight and gate that are there
  static variable_list forward(AutogradContext* ctx, at::TensorList given, const Seed& seed, unsigned which,
                               const c10::intrusive_ptr<Residual>& r) {
    const c10::DeviceGuard guard(given[0].device());
    Parts t;
    for (int i = 0, j = 0; i < 5; ++i)
      if (which >> i & 1) t[i] = whole(given[j++]);
    t[5] = seed.t;
    Tensor out[3];
    residual_forward(t, *r, out, true);
    variable_list saved;
    for (const Tensor& v : t)
      if (v.defined()) saved.push_back(v);
    saved.push_back(out[2]);
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["args"] = c10::IValue::make_capsule(r);
    ctx->saved_data["which"] = (int64_t)(which | (seed.t.defined() ? 32u : 0u));
    ctx->set_materialize_grads(false);
    if (!t[2].defined()) return {out[0]};
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t which = ctx->saved_data["which"].toInt();
    const auto r = c10::static_intrusive_pointer_cast<Residual>(ctx->saved_data["args"].toCapsule());
    Parts t;
    for (int i = 0, j = 0; i < 6; ++i)
      if (which >> i & 1) t[i] = saved[j++];
    for (const Tensor& g : grads) plain_gradient("residual_norm", g);
    const c10::DeviceGuard guard(t[0].device());
    const Tensor dh = whole(grads[0]), dy = grads.size() > 1 ? whole(grads[1]) : Tensor();
    Tensor out[5];
    if (r->a.rows == 0) {
      for (int i = 0, j = 0; i < 5; ++i)
        if (which >> i & 1 && ctx->needs_input_grad(j++)) out[i] = at::zeros_like(t[i]);
    } else if (dh.defined() || dy.defined()) {
      const at::NoGradGuard off;
      for (int i = 0, j = 0; i < 5; ++i)
        if (which >> i & 1 && ctx->needs_input_grad(j++)) out[i] = at::empty_like(t[i]);
      ngdn_residual_args a = r->a;
      point(a, t);
      a.rstd_h = static_cast<float*>(raw_out(saved.back()));
      a.rstd_b = a.rstd_h + a.rows;
      a.dh = raw(dh); a.dy = raw(dy);
      a.dx = raw_out(out[0]); a.dbranch = raw_out(out[1]); a.dweight = raw_out(out[2]); a.dpost_weight = raw_out(out[3]);
      a.dgate = raw_out(out[4]);
      const Tensor ws = at::empty({ngdn_residual_norm_ws(&a)}, t[0].options().dtype(at::kFloat));
      a.ws = static_cast<float*>(raw_out(ws));
      done(ngdn_residual_norm_bwd(&a, stream(t[0])), "ngdn_residual_norm_bwd");
    }
    if (at::GradMode::is_enabled()) {
      // a graph of the gradient: differentiable once, so a second time raises
      variable_list some;
      for (Tensor& g : out)
        if (g.defined()) { g = g.detach(); g.set_requires_grad(true); some.push_back(g); }
      const auto once = std::make_shared<torch::autograd::DelayedError>(
          "residual_norm: its gradient cannot be differentiated again", (int64_t)some.size());
      some = (*once)(std::move(some));
      size_t i = 0;
      for (Tensor& g : out)
        if (g.defined()) g = some[i++];
    }
    variable_list result;
    for (int i = 0; i < 5; ++i)
      if (which >> i & 1) result.push_back(out[i]);
    result.resize(result.size() + 3);       // the seed, which, r
    return result;
  }
};

// which values share one of the gate's; seq: the rows that share a row of it
int gate_kind(const Tensor& x, const Tensor& g, int64_t& seq) {
  const int64_t n = x.dim(), D = x.size(-1);
  if (g.dim() == 1 && g.size(0) == D) return 1;
  if (g.dim() == n) {
    if (g.sizes() == x.sizes()) return 4;
    if (n > 1 && g.size(-1) == 1 && g.sizes().slice(0, n - 1) == x.sizes().slice(0, n - 1)) return 3;
    if (g.size(-1) == D) {
      int64_t i = 0, groups = 1;
      while (i < n - 1 && g.size(i) == x.size(i)) groups *= g.size(i++);
      seq = 1;
      bool ones = true;
      for (int64_t j = i; j < n - 1; ++j) { ones = ones && g.size(j) == 1; seq *= x.size(j); }
      if (ones) return groups == 1 ? 1 : 2;
    }
  }
  refuse("residual_norm: gate " + shape(g) + " for x " + shape(x) +
         " ([D]; x's shape, its last or some of the ones before it 1)");
}

py::object residual_norm(const Tensor& x0, const Tensor& branch0, const Optional& weight0, const Optional& post0,
                         const Optional& gate0, double residual_scale, double branch_scale, double p,
                         const py::object& seed, const py::object& offset, double eps,
                         c10::optional<at::ScalarType> type) {
  const char* name = "residual_norm";
  if (x0.dim() < 1 || x0.sizes() != branch0.sizes())
    refuse("residual_norm: x " + shape(x0) + ", branch " + shape(branch0) + " (one shape, [..., D])");
  const int64_t D = x0.size(-1);
  if (D < 1 || D > 16384) refuse("residual_norm: rows of " + std::to_string(D) + " (1 to 16384)");
  const Tensor given_[] = {x0, branch0, given(weight0), given(post0), given(gate0)};
  const char* names[] = {"x", "branch", "weight", "post_weight", "gate"};
  for (int i = 0; i < 5; ++i) {
    const Tensor& t = given_[i];
    if (!t.defined()) continue;
    check_floats(name, names[i], t);
    if ((i == 2 || i == 3) && (t.dim() != 1 || t.size(0) != D))
      refuse(std::string(name) + ": " + names[i] + " " + shape(t) + " for x " + shape(x0));
  }
  const Stream s = stream_from(name, p, seed, offset);
  if (!(eps >= 0)) refuse("residual_norm: eps " + std::to_string(eps));
  const at::ScalarType h_type = x0.scalar_type(), y_type = type.value_or(h_type);
  if (y_type != at::kBFloat16 && y_type != at::kFloat && y_type != at::kHalf)
    refuse(std::string(name) + ": out_dtype " + c10::toString(y_type) + " (bf16, fp16 or fp32)");
  const auto r = c10::make_intrusive<Residual>();
  ngdn_residual_args& a = r->a;
  a.D = (int32_t)D;
  a.rows = x0.numel() / D;
  a.gate_kind = given_[4].defined() ? gate_kind(x0, given_[4], a.seq) : 0;
  for (const Tensor& t : given_)
    if (t.defined()) on_gpu(name, t, x0);
  if (s.seed_tensor.defined()) on_gpu(name, s.seed_tensor, x0);
  // the kernels' types: bf16 throughout, or an fp32 stream with any of the two
  Tensor x = widened(x0), branch = widened(branch0);
  r->y_type = y_type == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
  if (x.scalar_type() == at::kBFloat16 && (branch.scalar_type() != at::kBFloat16 || r->y_type != at::kBFloat16))
    x = x.to(at::kFloat);
  const Parts t{x, branch, widened(given_[2]), widened(given_[3]), widened(given_[4]),
                s.threshold ? s.seed_tensor : Tensor()};
  const auto kind = [](const Tensor& t) { return t.defined() ? code(t) : NGDN_F32; };
  a.x_dtype = code(x); a.branch_dtype = code(branch);
  a.y_dtype = r->y_type == at::kBFloat16 ? NGDN_BF16 : NGDN_F32;
  if (!t[2].defined()) a.y_dtype = a.x_dtype;
  a.w_dtype = kind(t[2]); a.pw_dtype = kind(t[3]); a.gate_dtype = kind(t[4]);
  a.residual_scale = (float)residual_scale; a.branch_scale = (float)branch_scale; a.eps = (float)eps;
  a.threshold = s.threshold; a.keep = s.keep(); a.seed = s.seed; a.offset = s.offset;
  Tensor out[3];
  auto free = std::make_unique<py::gil_scoped_release>();        // a launch may wait for room in the queue
  if (wants_grad({t[0], t[1], t[2], t[3], t[4]})) {
    std::vector<Tensor> there;
    unsigned which = 0;
    for (int i = 0; i < 5; ++i)
      if (t[i].defined()) { there.push_back(t[i]); which |= 1u << i; }
    const variable_list v = ResidualFn::apply(at::TensorList(there), Seed{t[5]}, which, r);
    out[0] = v[0];
    if (t[2].defined()) out[1] = v[1];
  } else {
    no_tangents(name, {t[0], t[1], t[2], t[3], t[4]});
    const at::NoGradGuard off;
    const c10::DeviceGuard guard(x0.device());
    residual_forward(whole(t), *r, out, false);
  }
  if (out[0].scalar_type() != h_type) out[0] = out[0].to(h_type);
  if (t[2].defined() && out[1].scalar_type() != y_type) out[1] = out[1].to(y_type);
  free.reset();
  if (!t[2].defined()) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

// a setting of the sampler: a number, or one a row
struct Setting {
  Tensor rows;
  double value = 0;
  Setting(const char* which, const py::object& v, const Tensor& u, bool whole_number, double low, double high) {
    if (THPVariable_Check(v.ptr())) {
      rows = THPVariable_Unpack(v.ptr()).detach();
      const auto t = rows.scalar_type();
      if (whole_number ? t != at::kInt && t != at::kLong : !floats(rows) && t != at::kDouble)
        refuse(std::string("sample_tokens: ") + which + " is " + c10::toString(t));
      if (rows.dim() != 0 && rows.sizes() != u.sizes())
        refuse(std::string("sample_tokens: ") + which + " " + shape(rows) + " for u " + shape(u));
      return;
    }
    if (whole_number) {
      if (!PyIndex_Check(v.ptr())) refuse(std::string("sample_tokens: ") + which + " must be an integer");
      const py::object i = py::reinterpret_steal<py::object>(PyNumber_Index(v.ptr()));
      if (!i) throw py::error_already_set();
      int over = 0;
      const long long n = PyLong_AsLongLongAndOverflow(i.ptr(), &over);
      value = over ? (over > 0 ? 1e9 : 0) : (double)(n > 1000000000 ? 1000000000 : n < 0 ? 0 : n);
      return;
    }
    value = PyFloat_AsDouble(v.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    if (!(value >= low && value <= high))
      refuse(std::string("sample_tokens: ") + which + " " + std::to_string(value) + " outside its range");
  }
  // its values as the kernel reads them: fp32 (top_k as it is), one a row
  const void* ptr(const Tensor& u, bool whole_number) {
    if (!rows.defined()) return nullptr;
    if (!whole_number && rows.scalar_type() != at::kFloat) rows = rows.to(at::kFloat);
    rows = whole(rows.dim() == 0 ? rows.expand(u.sizes()) : rows);
    return raw(rows);
  }
};

Tensor sample_tokens(const Tensor& logits0, const Tensor& u0, const py::object& temperature, const py::object& top_k,
                     const py::object& top_p, const py::object& min_p) {
  const char* name = "sample_tokens";
  check_floats(name, "logits", logits0);
  if (logits0.dim() < 1 || logits0.size(-1) < 1 || logits0.size(-1) > 1 << 20)
    refuse("sample_tokens: logits " + shape(logits0) + " ([..., V], 1 <= V <= 2^20)");
  if (u0.sizes() != logits0.sizes().slice(0, logits0.dim() - 1))
    refuse("sample_tokens: u " + shape(u0) + " for logits " + shape(logits0));
  if (u0.scalar_type() != at::kFloat && u0.scalar_type() != at::kDouble)
    refuse(std::string("sample_tokens: u is ") + c10::toString(u0.scalar_type()) + " (fp32 or fp64)");
  Setting t("temperature", temperature, u0, false, 0, 3.4028234663852886e38), k("top_k", top_k, u0, true, 0, 0),
      p("top_p", top_p, u0, false, 0, 1), m("min_p", min_p, u0, false, 0, 1);
  on_gpu(name, logits0, logits0);
  for (const Tensor& v : {u0, t.rows, k.rows, p.rows, m.rows})
    if (v.defined()) on_gpu(name, v, logits0);
  const py::gil_scoped_release free;
  const at::NoGradGuard off;
  const c10::DeviceGuard guard(logits0.device());
  const Tensor u = whole(u0.detach());
  Tensor logits = widened(logits0.detach()).resolve_neg();
  const int64_t V = logits.size(-1);
  int64_t step = V;
  if (logits.dim() == 2 && (logits.stride(1) == 1 || V == 1)) step = logits.stride(0);
  else logits = whole(logits);
  Tensor token = at::empty(u.sizes(), u.options().dtype(at::kLong));
  ngdn_sample_args a{};
  a.rows = u.numel(); a.stride = step; a.V = (int32_t)V;
  a.u_wide = u.scalar_type() == at::kDouble;
  a.temperature = (float)t.value; a.top_p = (float)p.value; a.min_p = (float)m.value; a.top_k = (int64_t)k.value;
  a.temperature_ptr = static_cast<const float*>(t.ptr(u, false));
  a.top_p_ptr = static_cast<const float*>(p.ptr(u, false));
  a.min_p_ptr = static_cast<const float*>(m.ptr(u, false));
  a.top_k_ptr = k.ptr(u, true);
  a.top_k_wide = k.rows.defined() && k.rows.scalar_type() == at::kLong;
  a.logits = raw(logits); a.u = raw(u);
  a.token = static_cast<int64_t*>(raw_out(token));
  done(ngdn_sample(code(logits), &a, stream(logits)), "ngdn_sample");
  return token;
}

// a failed call as _lib.NgdnError
template <typename F>
auto call(F f) -> decltype(f()) {
  try {
    return f();
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
  static PyTypeObject drop_fn, residual_fn;
  torch::autograd::_initFunctionPyTypeObject(drop_fn, "_DropoutFnBackward", nullptr, nullptr);
  torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<DropoutFn>), &drop_fn);
  torch::autograd::_initFunctionPyTypeObject(residual_fn, "_ResidualNormFnBackward", nullptr, nullptr);
  torch::autograd::registerCppFunction(typeid(torch::autograd::CppNode<ResidualFn>), &residual_fn);
  m.attr("version") = NGDN_VERSION;
  m.def("setup", [](py::object grad, py::object error) {
    python_grad = new py::object(std::move(grad));
    ngdn_error = new py::object(std::move(error));
  });
  m.def("embedding", &embedding);
  m.def("dropout", [](const Tensor& x, double p, const py::object& seed, const py::object& offset) {
    return call([&] { return dropout(x, p, seed, offset); });
  });
  m.def("residual_norm", [](const Tensor& x, const Tensor& branch, const Optional& weight, const Optional& post,
                            const Optional& gate, double rs, double bs, double p, const py::object& seed,
                            const py::object& offset, double eps, c10::optional<at::ScalarType> type) {
    return call([&] { return residual_norm(x, branch, weight, post, gate, rs, bs, p, seed, offset, eps, type); });
  });
  m.def("sample_tokens", [](const Tensor& logits, const Tensor& u, const py::object& t, const py::object& k,
                            const py::object& p, const py::object& least) {
    return call([&] { return sample_tokens(logits, u, t, k, p, least); });
  });
}
