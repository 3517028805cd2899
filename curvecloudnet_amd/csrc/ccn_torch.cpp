// The operators whose host side would cost more than their kernels, bound to torch in C++: argument checks, output tensors, tables of
// hundreds of tensors and the autograd node of the log-probabilities.  A node in Python has its device thread and the caller
// hand the interpreter's lock to and fro (forward and backward of 1000 x 20 logits: 117 us on the host, of which the kernels need 10).
// The kernels are reached through the C ABI of libccn_hip.so (include/ccn_hip.h), whose addresses `bind` is given once.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <cmath>

#include "../../include/ccn_hip.h"

namespace {

using at::Tensor;

struct Entries {
  decltype(&ccn_last_error) last_error;
  decltype(&ccn_logprob_workspace_bytes) logprob_workspace_bytes;
  decltype(&ccn_logprob_fwd) logprob_fwd;
  decltype(&ccn_logprob_bwd) logprob_bwd;
  decltype(&ccn_grad_norm_workspace_bytes) grad_norm_workspace_bytes;
  decltype(&ccn_grad_norm) grad_norm;
  decltype(&ccn_grad_clip) grad_clip;
  decltype(&ccn_adam_clip) adam_clip;
} entry;

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& addresses) {
  take(entry.last_error, addresses, "ccn_last_error");
  take(entry.logprob_workspace_bytes, addresses, "ccn_logprob_workspace_bytes");
  take(entry.logprob_fwd, addresses, "ccn_logprob_fwd");
  take(entry.logprob_bwd, addresses, "ccn_logprob_bwd");
  take(entry.grad_norm_workspace_bytes, addresses, "ccn_grad_norm_workspace_bytes");
  take(entry.grad_norm, addresses, "ccn_grad_norm");
  take(entry.grad_clip, addresses, "ccn_grad_clip");
  take(entry.adam_clip, addresses, "ccn_adam_clip");
}

// What _lib.call does around a launch (timing, the log of launches) is done there for these too, where it is asked for: `observer`
// gets the entry's name, its integer arguments, the values it works on and the launch itself.
std::atomic<bool> observed{false};
PyObject* observer = nullptr;               // (never freed: a backward pass may still be on its way there)

void observe(const py::object& f) {
  observed = false;
  if (f.is_none()) return;
  observer = f.inc_ref().ptr();
  observed = true;
}

template <typename F>
void launch(const char* name, std::initializer_list<int64_t> ints, int64_t work, const F& run) {
  int rc = 0;
  if (observed) {
    py::gil_scoped_acquire gil;
    py::reinterpret_borrow<py::object>(observer)(name, py::tuple(py::cast(std::vector<int64_t>(ints))), work,
                                                 py::cpp_function([&] { rc = run(); }));
  } else {
    rc = run();
  }
  TORCH_CHECK(rc == 0, "libccn_hip ", name, " failed (", rc, "): ", entry.last_error());
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

std::string name_of(at::ScalarType t) { return py::str(py::cast(t)); }

int code_of(at::ScalarType t) { return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1; }

void require_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "curvecloudnet_amd ops run on the GPU only (got a ", t.device().str(), " tensor); there is no CPU path");
}

// ---- log-probabilities

constexpr int64_t TOP_MAX = 64;

// A gradient as the kernels read it: the engine hands some down with their sign still to be turned (those of imaginary parts), which
// contiguous() leaves as it is.
Tensor settled(const Tensor& g) { return g.defined() ? g.resolve_neg() : g; }

// Logits (rows, C) as the kernels read them: columns adjacent, rows in order and apart.
Tensor rows_of(Tensor x) {
  if (x.is_neg()) x = x.resolve_neg();
  // (one row: its stride is never used, and torch may report any)
  if ((x.stride(1) != 1 && x.size(1) > 1) || (x.size(0) > 1 && x.stride(0) < x.size(1))) x = x.contiguous();
  return x;
}

template <typename T>
T* data(const Tensor& t) {
  return t.defined() ? t.mutable_data_ptr<T>() : nullptr;
}

struct Scored {
  Tensor logprob, entropy, best, index, stats;
};

// logits: (rows, C), the columns adjacent; target: int64, contiguous
Scored score(const Tensor& logits, const Tensor& target, int64_t top, int64_t ignore, bool with_stats) {
  const int64_t rows = logits.size(0), c = logits.size(1);
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(logits.device());
  c10::DeviceGuard guard(logits.device());
  Scored s;
  s.logprob = at::empty({rows}, f32);
  s.entropy = at::empty({rows}, f32);
  if (with_stats) s.stats = at::empty({rows, 2}, f32);
  if (top) {
    s.best = at::empty({rows, top}, f32);
    s.index = at::empty({rows, top}, f32.dtype(at::kLong));
  }
  if (rows == 0) return s;
  const int64_t bytes = (int64_t)entry.logprob_workspace_bytes(rows, c, (int)top);
  Tensor ws;
  if (bytes) ws = at::empty({bytes}, f32.dtype(at::kByte));
  const int code = code_of(logits.scalar_type());
  launch("logprob_fwd", {code, logits.stride(0), rows, c, ignore, top, bytes}, rows, [&] {
    return entry.logprob_fwd(logits.const_data_ptr(), code, logits.stride(0), target.const_data_ptr<int64_t>(), rows, c, ignore, (int)top,
                             data<float>(s.logprob), data<float>(s.entropy), data<float>(s.stats), data<float>(s.best),
                             data<int64_t>(s.index), data<uint8_t>(ws), (size_t)bytes, stream_of(logits));
  });
  return s;
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& target,
                                                int64_t top, int64_t ignore) {
    const Scored s = score(logits, target, top, ignore, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, target, s.index, s.stats, s.entropy});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["rows"] = logits.size(0);
    ctx->saved_data["classes"] = logits.size(1);
    ctx->saved_data["device"] = (int64_t)logits.get_device();
    if (!top) return {s.logprob, s.entropy};
    ctx->mark_non_differentiable({s.index});
    return {s.logprob, s.entropy, s.best, s.index};
  }

  static Tensor gradient(torch::autograd::AutogradContext* ctx, const torch::autograd::variable_list& grads) {
    const Tensor g_logprob = settled(grads[0]), g_entropy = settled(grads[1]);
    const Tensor g_top = grads.size() > 2 && grads[2].defined() ? settled(grads[2]).contiguous() : Tensor();
    const int64_t rows = ctx->saved_data["rows"].toInt(), c = ctx->saved_data["classes"].toInt();
    const int64_t device = ctx->saved_data["device"].toInt(), top = g_top.defined() ? g_top.size(1) : 0;
    // (a hook on saved tensors may have laid them out anew, and torch does not look at what it gives back)
    const auto saved = ctx->get_saved_variables();
    const auto kept = [&](size_t i, at::ScalarType type, at::IntArrayRef shape) {
      const Tensor& t = saved[i];
      TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.sizes() == shape && t.is_cuda() && t.get_device() == device &&
                      (t.scalar_type() == type || (i == 0 && code_of(t.scalar_type()) >= 0)),
                  "token_logprobs: a hook on saved tensors gave back another tensor than was saved");
      return i == 0 ? rows_of(t) : t.resolve_neg().contiguous();
    };
    const Tensor logits = kept(0, at::kFloat, {rows, c}), target = kept(1, at::kLong, {rows});
    const Tensor index = top ? kept(2, at::kLong, {rows, top}) : Tensor();
    const Tensor stats = kept(3, at::kFloat, {rows, 2}), entropy = kept(4, at::kFloat, {rows});
    const int64_t ignore = ctx->saved_data["ignore"].toInt(), per = logits.scalar_type() == at::kFloat ? 4 : 8;
    const int64_t ld = (c + per - 1) / per * per;            // rows start 16-byte aligned
    c10::DeviceGuard guard(logits.device());
    Tensor d = at::empty({rows, ld}, logits.options());
    if (ld != c) d = d.narrow(1, 0, c);
    if (rows == 0) return d;
    const int code = code_of(logits.scalar_type());
    const int64_t s1 = g_logprob.defined() ? g_logprob.stride(0) : 0, s2 = g_entropy.defined() ? g_entropy.stride(0) : 0;
    launch("logprob_bwd", {code, logits.stride(0), rows, c, ignore, top, s1, s2, ld}, rows, [&] {
      return entry.logprob_bwd(logits.const_data_ptr(), code, logits.stride(0), target.const_data_ptr<int64_t>(), rows, c, ignore,
                               (int)top, top ? data<int64_t>(index) : nullptr, data<float>(stats), data<float>(entropy),
                               data<float>(g_logprob), s1, data<float>(g_entropy), s2, data<float>(g_top), d.mutable_data_ptr(), ld,
                               stream_of(logits));
    });
    return d;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return {gradient(ctx, grads), Tensor(), Tensor(), Tensor()};
    // create_graph: what the gradient depends on is not followed, and whoever asks for it is told so
    Tensor d;
    {
      at::NoGradGuard off;
      d = gradient(ctx, grads).detach();
    }
    d.requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("token_logprobs: its gradient cannot be differentiated again", 1);
    return {(*error)({d})[0], Tensor(), Tensor(), Tensor()};
  }
};

py::tuple token_logprobs(const Tensor& logits, const Tensor& target, int64_t top, int64_t ignore) {
  TORCH_CHECK_TYPE(code_of(logits.scalar_type()) >= 0, "token_logprobs: logits are ", name_of(logits.scalar_type()),
                   "; fp32, bf16 or fp16 is wanted");
  TORCH_CHECK_TYPE(target.scalar_type() == at::kLong || target.scalar_type() == at::kInt, "token_logprobs: target is ",
                   name_of(target.scalar_type()), "; int64 or int32 is wanted");
  TORCH_CHECK_VALUE(logits.dim() > 0 && logits.size(-1) > 0 && logits.size(-1) < (int64_t)1 << 30, "token_logprobs: logits of shape ",
                    logits.sizes(), " have no classes, or too many");
  const int64_t c = logits.size(-1), rows = target.numel();
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(target.sizes() == shape, "token_logprobs: logits of shape ", logits.sizes(), " want a target of shape ", shape, ", got ",
                    target.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= std::min(TOP_MAX, c), "token_logprobs: top=", top, "; 0 to ", std::min(TOP_MAX, c), " is wanted");
  TORCH_CHECK_VALUE(rows < (int64_t)1 << 31, "token_logprobs: ", rows, " rows");
  require_gpu(logits);
  require_gpu(target);
  TORCH_CHECK_VALUE(logits.device() == target.device(), "token_logprobs: logits on ", logits.device().str(), ", target on ",
                    target.device().str());
  const bool flat = logits.dim() == 2;
  const Tensor x = rows_of(flat ? logits : logits.reshape({rows, c}));
  Tensor t = target.is_neg() ? target.resolve_neg() : target;
  if (!flat || t.scalar_type() != at::kLong || !t.is_contiguous()) t = t.reshape({rows}).to(at::kLong).contiguous();
  Tensor logprob, entropy, best, index;
  // (a tangent of forward mode goes the same way: the node refuses it)
  if ((logits.requires_grad() && at::GradMode::is_enabled()) || logits._fw_grad(0).defined()) {
    const auto out = TokenLogProbs::apply(x, t, top, ignore);
    logprob = out[0];
    entropy = out[1];
    if (top) {
      best = out[2];
      index = out[3];
    }
  } else {
    Scored s = score(x, t, top, ignore, false);
    logprob = s.logprob;
    entropy = s.entropy;
    best = s.best;
    index = s.index;
  }
  if (!flat) {
    logprob = logprob.view(shape);
    entropy = entropy.view(shape);
    if (top) {
      auto wide = shape.vec();
      wide.push_back(top);
      best = best.view(wide);
      index = index.view(wide);
    }
  }
  if (!top) return py::make_tuple(logprob, entropy, py::none(), py::none());
  return py::make_tuple(logprob, entropy, best, index);
}

// ---- the norm of many gradients

// Addresses, sizes and types of tensors of one GPU, each of which fills one run of memory.
struct Table {
  std::vector<const void*> at;
  std::vector<int64_t> size;
  std::vector<int32_t> code;
  int64_t total = 0;
  Tensor one;
  int64_t n() const { return (int64_t)at.size(); }
};

Table table_of(const std::vector<Tensor>& tensors, const char* who, bool writes) {
  Table t;
  t.at.reserve(tensors.size());
  t.size.reserve(tensors.size());
  t.code.reserve(tensors.size());
  for (const Tensor& x : tensors) {
    c10::TensorImpl* const impl = x.unsafeGetTensorImpl();
    TORCH_CHECK_TYPE(impl->layout() == at::kStrided, who, ": sparse tensors are not built");
    const int code = code_of(x.scalar_type());
    TORCH_CHECK_TYPE(code >= 0, who, ": ", name_of(x.scalar_type()), "; fp32, bf16 or fp16 is wanted");
    TORCH_CHECK_VALUE(impl->is_non_overlapping_and_dense(), who, ": a tensor of strides ", x.strides(), " does not fill its memory");
    require_gpu(x);
    TORCH_CHECK_VALUE(impl->device() == tensors[0].device(), who, ": tensors on ", tensors[0].device().str(), " and ", x.device().str());
    const int64_t size = impl->numel();
    t.at.push_back(writes ? impl->mutable_data() : impl->data());
    t.size.push_back(size);
    t.code.push_back(code);
    t.total += size;
  }
  t.one = tensors[0];
  return t;
}

// ws and norm of a call, on the current device
struct NormOut {
  c10::DeviceGuard guard;
  int64_t bytes;
  Tensor ws, norm;
  NormOut(const Table& t)
      : guard(t.one.device()), bytes((int64_t)entry.grad_norm_workspace_bytes(t.n())),
        ws(at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(t.one.device()))),
        norm(at::empty({}, at::TensorOptions().dtype(at::kFloat).device(t.one.device()))) {}
};

void moved(const std::vector<Tensor>& tensors) {             // written behind torch's back: as an in-place operation
  for (const Tensor& t : tensors)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The i-th of a list; hundreds are looked at in place, without one Python object or count of references more than it takes.
const Tensor& tensor_at(const py::list& list, size_t i, const char* who) {
  PyObject* const o = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
  TORCH_CHECK_TYPE(THPVariable_Check(o), who, ": ", Py_TYPE(o)->tp_name, " is no tensor");
  return THPVariable_Unpack(o);
}

std::vector<Tensor> tensors_of(const py::list& list, const char* who) {
  std::vector<Tensor> tensors;
  tensors.reserve(list.size());
  for (size_t i = 0; i < list.size(); ++i) tensors.push_back(tensor_at(list, i, who));
  return tensors;
}

Tensor grad_norm(const py::list& list, int kind) {
  const std::vector<Tensor> tensors = tensors_of(list, "grad_norm");
  const Table t = table_of(tensors, "grad_norm", false);
  NormOut o(t);
  launch("grad_norm", {t.n(), kind, o.bytes}, t.total, [&] {
    return entry.grad_norm(t.at.data(), t.size.data(), t.code.data(), t.n(), kind, o.ws.mutable_data_ptr(), (size_t)o.bytes,
                           o.norm.mutable_data_ptr<float>(), stream_of(t.one));
  });
  return o.norm;
}

// The gradients of `parameters`, those that have one.
std::vector<Tensor> grads_of(const py::list& parameters) {
  std::vector<Tensor> grads;
  grads.reserve(parameters.size());
  for (size_t i = 0; i < parameters.size(); ++i) {
    const Tensor& g = tensor_at(parameters, i, "clip_grad_norm_").unsafeGetTensorImpl()->grad();
    if (g.defined()) grads.push_back(g);
  }
  return grads;
}

// None where no parameter has a gradient.
py::object clip_grad_norm(const py::list& parameters, int kind, double max_norm) {
  const std::vector<Tensor> grads = grads_of(parameters);
  if (grads.empty()) return py::none();
  const Table t = table_of(grads, "clip_grad_norm_", true);
  NormOut o(t);
  launch("grad_clip", {t.n(), kind, o.bytes}, t.total, [&] {
    return entry.grad_clip(const_cast<void* const*>(t.at.data()), t.size.data(), t.code.data(), t.n(), kind, max_norm,
                           o.ws.mutable_data_ptr(), (size_t)o.bytes, o.norm.mutable_data_ptr<float>(), stream_of(t.one));
  });
  moved(grads);
  return py::cast(o.norm);
}

// ---- the update

py::object adam_step(const py::list& of_params, const py::list& of_grads, const py::list& of_exp_avgs, const py::list& of_exp_avg_sqs,
                     int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay, std::optional<double> max_norm) {
  const std::vector<Tensor> params = tensors_of(of_params, "adam_step_"), grads = tensors_of(of_grads, "adam_step_"),
                            exp_avgs = tensors_of(of_exp_avgs, "adam_step_"), exp_avg_sqs = tensors_of(of_exp_avg_sqs, "adam_step_");
  const std::vector<Tensor>* lists[4] = {&params, &grads, &exp_avgs, &exp_avg_sqs};
  for (int k = 1; k < 4; ++k)
    TORCH_CHECK_VALUE(lists[k]->size() == params.size(), "adam_step_: ", params.size(), " parameters, ", grads.size(), " gradients, ",
                      exp_avgs.size(), " and ", exp_avg_sqs.size(), " moments");
  for (const auto* v : lists)
    for (size_t i = 0; i < v->size(); ++i) {
      const Tensor& t = (*v)[i];
      TORCH_CHECK_TYPE(t.layout() == at::kStrided && t.scalar_type() == at::kFloat, "adam_step_: fp32 tensors are wanted");
      TORCH_CHECK_VALUE(t.numel() == params[i].numel() && t.is_contiguous(),
                        "adam_step_: the tensors of a parameter are contiguous and of one size");
      TORCH_CHECK_VALUE(!t.is_neg(), "adam_step_: a tensor whose sign is still to be turned");
    }
  for (const auto* v : lists)
    for (const Tensor& t : *v) {
      require_gpu(t);
      TORCH_CHECK_VALUE(t.device() == params[0].device(), "adam_step_: tensors on ", params[0].device().str(), " and ", t.device().str());
      TORCH_CHECK_VALUE((uintptr_t)t.const_data_ptr() % 16 == 0, "adam_step_: a tensor does not start at a multiple of 16 bytes");
    }
  Table t[4];
  for (int k = 0; k < 4; ++k) t[k] = table_of(*lists[k], "adam_step_", k != 1);
  const auto run = [&](double bound, void* ws, int64_t bytes, float* norm) {
    launch("adam_clip", {t[1].n(), step, bytes}, t[1].total, [&] {
      return entry.adam_clip((float* const*)t[0].at.data(), (const float* const*)t[1].at.data(), (float* const*)t[2].at.data(),
                             (float* const*)t[3].at.data(), t[1].size.data(), t[1].n(), lr, beta1, beta2, eps, weight_decay, step, bound,
                             ws, (size_t)bytes, norm, stream_of(t[1].one));
    });
  };
  py::object norm = py::none();
  if (max_norm) {
    NormOut o(t[1]);
    run(*max_norm, o.ws.mutable_data_ptr(), o.bytes, o.norm.mutable_data_ptr<float>());
    norm = py::cast(o.norm);
  } else {
    c10::DeviceGuard guard(t[1].one.device());
    run(INFINITY, nullptr, 0, nullptr);
  }
  moved(params);
  moved(exp_avgs);
  moved(exp_avg_sqs);
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", torch::wrap_pybind_function(bind));
  m.def("observe", torch::wrap_pybind_function(observe));
  m.def("token_logprobs", torch::wrap_pybind_function(token_logprobs));
  m.def("grad_norm", torch::wrap_pybind_function(grad_norm));
  m.def("grads_of", torch::wrap_pybind_function(grads_of));
  m.def("clip_grad_norm", torch::wrap_pybind_function(clip_grad_norm));
  m.def("adam_step", torch::wrap_pybind_function(adam_step));
}
