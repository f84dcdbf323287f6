// class_scores.cpp -- torch's side of the losses over rows of class scores:
// argument checks, outputs and the autograd nodes around the C entries of
// libb2ocl.so (b2_token_log_probs and the others of that section).
//
// These losses take the GPU microseconds where tokens are few, and a node
// written in Python costs the host over 50 us, most of it for the way of the
// gradient through the interpreter; here a loss with its gradient takes little
// more than torch's engine itself.  The entries' addresses and the package's
// error types come from opencl_tf/_library.py, so that both go through the one
// library that is loaded.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/custom_class.h>
#include <torch/extension.h>

#include <cstring>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "b2_opencl_tf.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

namespace {

struct Entries {
  decltype(&b2_token_log_probs) token_log_probs;
  decltype(&b2_token_log_probs_grad) token_log_probs_grad;
  decltype(&b2_distillation_loss) distillation_loss;
  decltype(&b2_distillation_loss_grad) distillation_loss_grad;
  decltype(&b2_preference_loss) preference_loss;
  decltype(&b2_preference_loss_grad) preference_loss_grad;
  decltype(&b2_policy_loss) policy_loss;
  decltype(&b2_policy_loss_grad) policy_loss_grad;
  decltype(&b2_policy_loss_with_grad) policy_loss_with_grad;
} entries;
PyObject* invalid_argument = nullptr;  // errors.InvalidArgumentError
PyObject* raise_status = nullptr;      // raises the error of a status, with this thread's message

// ------------------------------------------------------------------ errors

[[noreturn]] void invalid(const std::string& message) {
  PyErr_SetString(invalid_argument, message.c_str());
  throw py::error_already_set();
}

// Calls a C entry on `t`'s device and torch's current stream of it.  With the
// GIL held (forward) the error is Python's at once; a node of the engine, which
// runs without it, hands it over to the thread that waits for the gradients.
template <class F, class... Args>
void call(bool in_engine, const Tensor& t, F entry, Args... args) {
  const auto device = t.device();
  int rc;
  {
    c10::cuda::CUDAGuard guard(device);
    const auto stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    if (in_engine) {
      rc = entry(stream, args...);
    } else {
      py::gil_scoped_release release;  // a launch may wait for room in its queue
      rc = entry(stream, args...);
    }
  }
  if (rc == B2_OK) return;
  if (!in_engine) {
    Py_XDECREF(PyObject_CallFunction(raise_status, "i", rc));
    throw py::error_already_set();
  }
  py::gil_scoped_acquire gil;
  Py_XDECREF(PyObject_CallFunction(raise_status, "i", rc));
  python_error error;
  error.persist();
  throw error;
}

// --------------------------------------------------------------- arguments

enum Types : unsigned { kF32 = 1, kF16 = 2, kBF16 = 4, kI32 = 8, kI64 = 16, kBool = 32, kU8 = 64 };
constexpr unsigned kFloats = kF32 | kF16 | kBF16, kInts = kI32 | kI64, kWeights = kF32 | kBool | kU8;

unsigned type_bit(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kF32;
    case at::kHalf: return kF16;
    case at::kBFloat16: return kBF16;
    case at::kInt: return kI32;
    case at::kLong: return kI64;
    case at::kBool: return kBool;
    case at::kByte: return kU8;
    default: return 0;
  }
}

std::string names_of(unsigned types) {
  const char* all[] = {"float32", "float16", "bfloat16", "int32", "int64", "bool", "uint8"};
  std::string s;
  for (unsigned i = 0; i < 7; ++i)
    if (types >> i & 1u) s += (s.empty() ? "" : ", ") + std::string(all[i]);
  return s;
}

std::string text(at::ScalarType t) { return c10::toString(t); }

std::string text(c10::IntArrayRef shape) {
  std::string s = "[";
  for (const int64_t n : shape) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
  return s + "]";
}

b2_dtype_t dtype_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? B2_FLOAT32 : t.scalar_type() == at::kHalf ? B2_FLOAT16 : B2_BFLOAT16;
}

const Tensor& on_cuda(py::handle h, const char* what) {
  if (!THPVariable_Check(h.ptr())) invalid(std::string(what) + " must be a torch tensor on a CUDA device");
  const Tensor& t = THPVariable_Unpack(h.ptr());
  if (!t.is_cuda()) invalid(std::string(what) + " must live on a CUDA device (this backend has no CPU path)");
  return t;
}

// The losses have no forward-mode derivative; a tangent is refused, not dropped.
const Tensor& no_tangent(const Tensor& t, const char* what) {
  if (t._fw_grad(0).defined())
    invalid(std::string(what) + " has a forward-mode tangent: the losses over class scores are differentiated backward");
  return t;
}

// A tensor of one of the types on `like`'s device, of the given shape; contiguous.
Tensor same(py::handle h, const char* what, c10::IntArrayRef shape, const Tensor& like, unsigned types) {
  const Tensor& t = on_cuda(h, what);
  if (!(type_bit(t) & types))
    invalid(std::string(what) + " must be " + names_of(types) + ", got " + text(t.scalar_type()));
  if (t.sizes() != shape)
    invalid(std::string(what) + " must have shape " + text(shape) + ", got " + text(t.sizes()));
  if (t.device() != like.device())
    invalid(std::string(what) + " must live on " + like.device().str() + ", got " + t.device().str());
  return t.contiguous();
}

Tensor opt_same(py::handle h, const char* what, c10::IntArrayRef shape, const Tensor& like, unsigned types) {
  return h.is_none() ? Tensor() : same(h, what, shape, like, types);
}

Tensor opt_scalar(py::handle h, const char* what, const Tensor& like) {
  if (h.is_none()) return Tensor();
  const Tensor& t = on_cuda(h, what);
  if (t.scalar_type() != at::kFloat || t.numel() != 1 || t.device() != like.device())
    invalid(std::string(what) + " must be a float32 scalar on " + like.device().str());
  return t;
}

// Scores as rows: read in place where the leading axes fold into two strides.
struct Rows {
  Tensor x;
  b2_logits_t view;
  const b2_logits_t* operator&() const { return &view; }
};

std::optional<b2_logits_t> folded(const Tensor& t) {
  const int64_t classes = t.size(-1);
  b2_logits_t v{t.data_ptr(), dtype_of(t), 1, 1, classes, 0, 0};
  if (t.is_contiguous()) {
    v.inner = t.numel() / classes;
    v.inner_stride = classes;
    return v;
  }
  if (t.stride(-1) != 1 && classes != 1) return std::nullopt;
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};
  int axes = 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) {
    if (t.size(i) == 1) continue;
    if (axes > 0 && stride[axes - 1] == t.size(i) * t.stride(i)) {
      size[axes - 1] *= t.size(i);
      stride[axes - 1] = t.stride(i);
    } else if (axes == 2) {
      return std::nullopt;
    } else {
      size[axes] = t.size(i);
      stride[axes++] = t.stride(i);
    }
  }
  const int last = axes == 2 ? 1 : 0;
  v.inner = size[last];
  v.inner_stride = stride[last];
  if (axes == 2) {
    v.outer = size[0];
    v.outer_stride = stride[0];
  }
  return v;
}

Rows rows_of(const Tensor& t) {
  if (auto v = folded(t)) return Rows{t, *v};
  Tensor x = t.contiguous();
  return Rows{x, *folded(x)};
}

const Tensor& scores(py::handle h) {
  const Tensor& t = on_cuda(h, "logits");
  if (!(type_bit(t) & kFloats)) invalid("logits must be " + names_of(kFloats) + ", got " + text(t.scalar_type()));
  if (t.dim() < 1 || t.size(-1) < 1) invalid("logits must be [..., classes] with at least one class");
  return no_tangent(t, "logits");
}

c10::IntArrayRef leading(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

int64_t rows_in(const Tensor& t) { return t.numel() / t.size(-1); }

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(data(t)); }
int width(const Tensor& t) { return t.defined() ? static_cast<int>(t.element_size()) : 0; }

Tensor new_f32(const Tensor& like, c10::IntArrayRef shape) {
  return at::empty(shape, like.options().dtype(at::kFloat));
}
Tensor new_dense(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// ------------------------------------------------------------------- nodes

// The losses are differentiable once: where a backward pass is itself recorded,
// its result gets a node that says so if it is gone through, with an edge to the
// loss's scores or log-probabilities and one to the upstream gradient, on which the
// result depends as well.
Tensor once(Tensor grad, const torch::autograd::Edge& input, const Tensor& upstream) {
  torch::autograd::edge_list edges{input};
  if (upstream.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(upstream));
  const auto node = std::make_shared<torch::autograd::Error>(
      "the gradient of a loss over class scores is differentiable once", std::move(edges));
  torch::autograd::create_gradient_edge(grad, node);
  return grad;
}

Tensor once(const Tensor& grad, const Tensor& input, const Tensor& upstream) {
  return at::GradMode::is_enabled() ? once(grad, torch::autograd::impl::gradient_edge(input), upstream) : grad;
}

// What a gradient needs of log-probabilities that need not be kept for it.
struct Origin : torch::CustomClassHolder {
  explicit Origin(const Tensor& t) : edge(torch::autograd::impl::gradient_edge(t)), shape(t.sizes().vec()) {}
  torch::autograd::Edge edge;
  std::vector<int64_t> shape;

  static void keep(AutogradContext* ctx, const Tensor& t) {
    ctx->saved_data["origin"] = c10::IValue::make_capsule(c10::make_intrusive<Origin>(t));
  }
  static c10::intrusive_ptr<Origin> of(AutogradContext* ctx) {
    return c10::static_intrusive_pointer_cast<Origin>(ctx->saved_data["origin"].toCapsule());
  }
};

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static Tensor run(const Tensor& logits, const Tensor& targets, const Tensor& stats) {
    const Rows x = rows_of(logits);
    Tensor out = new_f32(logits, targets.sizes());
    call(false, logits, entries.token_log_probs, &x, targets.data_ptr(), width(targets), floats(out), floats(stats));
    return out;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor* targets) {
    Tensor stats = new_f32(logits, {targets->numel(), 2});
    Tensor out = run(logits, *targets, stats);
    ctx->save_for_backward({logits, *targets, stats});
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &targets = saved[1];
    Tensor out;
    {
      at::NoGradGuard quiet;
      const Rows x = rows_of(logits);
      const Tensor g = grads[0].contiguous();
      out = new_dense(logits);
      call(true, logits, entries.token_log_probs_grad, &x, targets.data_ptr(), width(targets), floats(saved[2]),
           floats(g), out.data_ptr());
    }
    return {once(out, logits, grads[0]), Tensor()};
  }
};

Tensor token_log_probs(py::handle logits, py::handle targets) {
  const Tensor& x = scores(logits);
  const Tensor t = same(targets, "targets", leading(x), x, kInts);
  return records(x) ? TokenLogProbs::apply(x, &t) : TokenLogProbs::run(x, t, Tensor());
}

struct Teacher {
  Tensor ids, y, weights;
  double temperature;
};

Teacher teacher_of(const Tensor& x, py::handle ids, py::handle y, py::handle weights, double temperature) {
  const Tensor& i = on_cuda(ids, "teacher_ids");
  if (i.dim() != x.dim() || leading(i) != leading(x))
    invalid("teacher_ids must be [..., entries] with the leading axes of logits " + text(x.sizes()) + ", got " +
            text(i.sizes()));
  Teacher t;
  t.ids = same(ids, "teacher_ids", i.sizes(), x, kInts);
  t.y = same(y, "teacher_logits", i.sizes(), x, kFloats);
  t.weights = opt_same(weights, "weights", leading(x), x, kWeights);
  t.temperature = temperature;
  return t;
}

struct Distillation : torch::autograd::Function<Distillation> {
  // stats: the rows' statistics, the sum of the weights and the call's workspace
  static Tensor run(const Tensor& logits, const Teacher& t, const Tensor& stats, const Tensor& grad_loss,
                    const Tensor& grad) {
    const Rows x = rows_of(logits);
    Tensor loss = new_f32(logits, {});
    call(false, logits, entries.distillation_loss, &x, t.ids.data_ptr(), width(t.ids), t.y.data_ptr(),
         static_cast<int>(dtype_of(t.y)), t.ids.size(-1), data(t.weights), width(t.weights), t.temperature,
         floats(loss), floats(stats), floats(grad_loss), data(grad));
    return loss;
  }
  static Tensor new_stats(const Tensor& logits) { return new_f32(logits, {4 * rows_in(logits) + 2}); }
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Teacher* t) {
    Tensor stats = new_stats(logits);
    Tensor loss = run(logits, *t, stats, Tensor(), Tensor());
    ctx->save_for_backward({logits, t->ids, t->y, t->weights, stats});
    ctx->saved_data["temperature"] = t->temperature;
    return loss;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &ids = saved[1], &y = saved[2], &weights = saved[3];
    Tensor out;
    {
      at::NoGradGuard quiet;
      const Rows x = rows_of(logits);
      out = new_dense(logits);
      call(true, logits, entries.distillation_loss_grad, &x, ids.data_ptr(), width(ids), y.data_ptr(),
           static_cast<int>(dtype_of(y)), ids.size(-1), data(weights), width(weights),
           ctx->saved_data["temperature"].toDouble(), floats(saved[4]), floats(grads[0]), out.data_ptr());
    }
    return {once(out, logits, grads[0]), Tensor()};
  }
};

Tensor distillation_loss(py::handle logits, py::handle ids, py::handle y, py::handle weights, double temperature) {
  const Tensor& x = scores(logits);
  const Teacher t = teacher_of(x, ids, y, weights, temperature);
  return records(x) ? Distillation::apply(x, &t)
                    : Distillation::run(x, t, Distillation::new_stats(x), Tensor(), Tensor());
}

std::tuple<Tensor, Tensor> distillation_loss_with_grad(py::handle logits, py::handle ids, py::handle y,
                                                       py::handle weights, double temperature, py::handle grad_loss) {
  at::NoGradGuard quiet;
  const Tensor& x = scores(logits);
  const Teacher t = teacher_of(x, ids, y, weights, temperature);
  const Tensor upstream = opt_scalar(grad_loss, "grad_loss", x);
  Tensor grad = new_dense(x);
  Tensor loss = Distillation::run(x, t, Distillation::new_stats(x), upstream, grad);
  return {loss, grad};
}

const Tensor& log_probs_of(py::handle h) {
  const Tensor& t = on_cuda(h, "log_probs");
  if (t.scalar_type() != at::kFloat) invalid("log_probs must be float32, got " + text(t.scalar_type()));
  return no_tangent(t, "log_probs");
}

struct Pairs {
  Tensor offsets, ref, mask;
  double beta, smoothing;
};

struct Preference : torch::autograd::Function<Preference> {
  static tensor_list run(const Tensor& log_probs, const Pairs& p, Tensor* slopes) {
    const Tensor lp = log_probs.contiguous();
    const int64_t sequences = p.offsets.numel() - 1;
    Tensor loss = new_f32(lp, {}), rewards = new_f32(lp, {sequences});
    *slopes = new_f32(lp, {sequences});
    call(false, lp, entries.preference_loss, floats(lp), floats(p.ref), data(p.mask), width(p.mask), lp.numel(),
         p.offsets.data_ptr(), width(p.offsets), sequences / 2, p.beta, p.smoothing, floats(loss), floats(rewards),
         floats(*slopes));
    return {loss, rewards};
  }
  static tensor_list forward(AutogradContext* ctx, const Tensor& log_probs, const Pairs* p) {
    Tensor slopes;
    tensor_list out = run(log_probs, *p, &slopes);
    ctx->save_for_backward({p->offsets, p->mask, slopes});
    Origin::keep(ctx, log_probs);
    ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &offsets = saved[0], &mask = saved[1], &slopes = saved[2];
    const auto origin = Origin::of(ctx);
    Tensor out;
    {
      at::NoGradGuard quiet;
      out = new_f32(slopes, origin->shape);
      call(true, out, entries.preference_loss_grad, floats(grads[0]), floats(slopes), data(mask), width(mask),
           out.numel(), offsets.data_ptr(), width(offsets), slopes.numel() / 2, floats(out));
    }
    return {at::GradMode::is_enabled() ? once(out, origin->edge, grads[0]) : out, Tensor()};
  }
};

std::tuple<Tensor, Tensor> preference_loss(py::handle log_probs, py::handle offsets, py::handle ref, py::handle mask,
                                           double beta, double smoothing) {
  const Tensor& lp = log_probs_of(log_probs);
  const Tensor& o = on_cuda(offsets, "offsets");
  if (o.dim() != 1 || o.numel() < 3 || o.numel() % 2 == 0)
    invalid("offsets must have 2 * pairs + 1 elements, pairs >= 1");
  const Pairs p{same(offsets, "offsets", o.sizes(), lp, kInts), opt_same(ref, "ref_log_probs", lp.sizes(), lp, kF32),
                opt_same(mask, "mask", lp.sizes(), lp, kWeights), beta, smoothing};
  Tensor slopes;
  const tensor_list out = records(lp) ? Preference::apply(lp, &p) : Preference::run(lp, p, &slopes);
  return {out[0], out[1]};
}

struct Tokens {
  Tensor old, advantages, ref, mask;
  double clip_low, clip_high, kl_coef;
};

Tokens tokens_of(const Tensor& like, c10::IntArrayRef shape, py::handle old, py::handle advantages, py::handle ref,
                 py::handle mask, double clip_low, double clip_high, double kl_coef) {
  return Tokens{same(old, "old_log_probs", shape, like, kF32),
                same(advantages, "advantages", shape, like, kF32),
                opt_same(ref, "ref_log_probs", shape, like, kF32),
                opt_same(mask, "mask", shape, like, kWeights),
                clip_low,
                clip_high,
                kl_coef};
}

struct Policy : torch::autograd::Function<Policy> {
  static tensor_list run(const Tensor& log_probs, const Tokens& t, const Tensor& slopes) {
    const Tensor lp = log_probs.contiguous();
    Tensor loss = new_f32(lp, {}), stats = new_f32(lp, {3});
    call(false, lp, entries.policy_loss, floats(lp), floats(t.old), floats(t.advantages), floats(t.ref), data(t.mask),
         width(t.mask), lp.numel(), t.clip_low, t.clip_high, t.kl_coef, floats(loss), floats(stats), floats(slopes));
    return {loss, stats};
  }
  static tensor_list forward(AutogradContext* ctx, const Tensor& log_probs, const Tokens* t) {
    Tensor slopes = new_dense(log_probs);
    tensor_list out = run(log_probs, *t, slopes);
    ctx->save_for_backward({out[1], slopes});
    Origin::keep(ctx, log_probs);
    ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor &stats = saved[0], &slopes = saved[1];
    const auto origin = Origin::of(ctx);
    Tensor out;
    {
      at::NoGradGuard quiet;
      out = new_dense(slopes);
      call(true, out, entries.policy_loss_grad, floats(grads[0]), floats(stats), floats(slopes), out.numel(),
           floats(out));
    }
    return {at::GradMode::is_enabled() ? once(out, origin->edge, grads[0]) : out, Tensor()};
  }
};

std::tuple<Tensor, Tensor> policy_loss(py::handle log_probs, py::handle old, py::handle advantages, py::handle ref,
                                       py::handle mask, double clip_low, double clip_high, double kl_coef) {
  const Tensor& lp = log_probs_of(log_probs);
  const Tokens t = tokens_of(lp, lp.sizes(), old, advantages, ref, mask, clip_low, clip_high, kl_coef);
  const tensor_list out = records(lp) ? Policy::apply(lp, &t) : Policy::run(lp, t, Tensor());
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor, Tensor> policy_loss_with_grad(py::handle logits, py::handle targets, py::handle old,
                                                         py::handle advantages, py::handle ref, py::handle mask,
                                                         double clip_low, double clip_high, double kl_coef,
                                                         py::handle grad_loss) {
  at::NoGradGuard quiet;
  const Tensor& x = scores(logits);
  const Tensor targets_t = same(targets, "targets", leading(x), x, kInts);
  const Tokens t = tokens_of(x, leading(x), old, advantages, ref, mask, clip_low, clip_high, kl_coef);
  const Tensor upstream = opt_scalar(grad_loss, "grad_loss", x);
  const Rows rows = rows_of(x);
  Tensor loss = new_f32(x, {}), stats = new_f32(x, {2}), grad = new_dense(x);
  call(false, x, entries.policy_loss_with_grad, &rows, targets_t.data_ptr(), width(targets_t), floats(t.old),
       floats(t.advantages), floats(t.ref), data(t.mask), width(t.mask), clip_low, clip_high, kl_coef, floats(upstream),
       floats(loss), floats(stats), grad.data_ptr());
  return {loss, stats, grad};
}

// ------------------------------------------------------------------ module

// addresses: of the entries, in the order of Entries.
void bind(const std::vector<uintptr_t>& addresses, py::object invalid_error, py::object raise) {
  TORCH_CHECK(addresses.size() * sizeof(uintptr_t) == sizeof(Entries), "one address for each entry");
  std::memcpy(&entries, addresses.data(), sizeof(Entries));
  invalid_argument = invalid_error.release().ptr();
  raise_status = raise.release().ptr();
}

// (outer, inner, classes, outer stride, inner stride) of scores that are read in place, None of others.
py::object fold(const Tensor& t) {
  const auto v = folded(t);
  if (!v) return py::none();
  return py::make_tuple(v->outer, v->inner, v->classes, v->outer_stride, v->inner_stride);
}

}  // namespace

PYBIND11_MODULE(_class_scores, m) {
  m.def("bind", &bind);
  m.def("fold", &fold);
  m.def("token_log_probs", &token_log_probs);
  m.def("distillation_loss", &distillation_loss);
  m.def("distillation_loss_with_grad", &distillation_loss_with_grad);
  m.def("preference_loss", &preference_loss);
  m.def("policy_loss", &policy_loss);
  m.def("policy_loss_with_grad", &policy_loss_with_grad);
}
