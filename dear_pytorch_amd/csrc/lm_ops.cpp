// Autograd nodes and launches of the language-model operators
// (layer_norm.hip, token_loss.hip). In C++ because at the sizes of a single
// token or a small batch the host's work, not the kernel, is the cost.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

int64_t dear_ln_blocks(int, int64_t, int);
int dear_ln_fwd(hipStream_t, int, int, int, const void*, int64_t, const void*,
                int64_t, const void*, const void*, void*, float*, int64_t, int,
                float);
int dear_ln_bwd(hipStream_t, int, int, int, const void*, int64_t, const void*,
                int64_t, const void*, int64_t, const void*, const float*,
                void*, void*, void*, void*, float*, int, int64_t, int);
int64_t dear_logprobs_work(int, int64_t, int, int);
int64_t dear_distill_work(int, int64_t, int);
int dear_logprobs_fwd(hipStream_t, int, const void*, int64_t, const int64_t*,
                      int64_t, int64_t, int, int, double, float*, float*,
                      float*, int64_t*, void*, void*);
int dear_logprobs_bwd(hipStream_t, int, const void*, int64_t, const int64_t*,
                      const int64_t*, const void*, const float*, const float*,
                      const float*, void*, int64_t, int, int, double);
int dear_distill_fwd(hipStream_t, int, bool, const void*, int64_t,
                     const int64_t*, const float*, int64_t, int, int, double,
                     float*, float*, void*, void*);
int dear_distill_bwd(hipStream_t, int, const void*, int64_t, const int64_t*,
                     const float*, const void*, const float*, void*, int64_t,
                     int, int, double);

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxWidth = int64_t(1) << 30;   // indices of a row are int
constexpr int64_t kMaxTop = 128;

void check_launch(int err) {
  TORCH_CHECK(err == 0, "HIP error: ", hipGetErrorString((hipError_t)err));
}

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      TORCH_CHECK_TYPE(false, name, " must be float32, bfloat16 or float16, "
                       "got ", t.scalar_type());
  }
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fdata(const Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}
int64_t* idata(const Tensor& t) {
  return t.defined() ? t.data_ptr<int64_t>() : nullptr;
}
using Maybe = c10::optional<Tensor>;
Tensor value(const Maybe& t) { return t ? *t : Tensor(); }

// A view whose elements are to be negated when they are read, as the imaginary
// part of a conjugate is: the kernels do not do that.
Tensor plain(const Tensor& t) {
  return t.defined() && t.is_neg() ? t.resolve_neg() : t;
}

// What torch would see of an operand and the kernels do not: to go on would
// lose it without a word.
void check_operands(std::initializer_list<Tensor> ts, const char* name) {
  // a trace would hold the results' allocation, and nothing that fills them
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() &&
          !c10::impl::TorchDispatchModeTLS::get_mode(
               c10::impl::TorchDispatchModeKey::PROXY)
               .has_value(),
      name, ": cannot be traced on a GPU");
  for (const auto& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(
        !t._fw_grad(/*level=*/0).defined(), name,
        ": forward-mode derivatives are not there on a GPU");
    // wrappers of other tensors, and fake ones
    TORCH_CHECK_TYPE(t.numel() == 0 || t.const_data_ptr() != nullptr, name,
                     ": an operand has no memory of its own");
  }
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// [rows, width] with a last stride of 1: a view where the strides allow one
Tensor as_rows(const Tensor& t, int64_t rows, int64_t width) {
  Tensor r = t.dim() == 2 ? t : t.reshape({rows, width});
  return width > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : c10::nullopt; }

// Gradients of a node that cannot be differentiated again: using them in a
// second backward pass raises, as torch's once_differentiable does.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)   // so that they get the node as their history
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " cannot be differentiated twice", grads.size());
  return (*node)(std::move(grads));
}

// Whether a node adds up a leaf's gradient on another stream than the current
// one, as it does while a graph that was made there lives.
bool accumulates_elsewhere(torch::autograd::Node* node) {
  if (!dynamic_cast<torch::autograd::AccumulateGrad*>(node)) return false;
  const auto stream = node->stream();
  if (!stream) return false;
  const c10::impl::VirtualGuardImpl guard(stream->device_type());
  return *stream != guard.getStream(stream->device());
}

// A captured backward pass cannot hand a gradient to a stream outside of the
// capture; the process would end where it tries to. To be called in a node's
// backward pass: looks at the leaves behind it that this pass has a gradient
// for.
void check_capture(hipStream_t stream, const char* name) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  check_launch((int)hipStreamIsCapturing(stream, &status));
  if (status == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  for (size_t i = 0; node && i < node->num_outputs(); ++i)
    TORCH_CHECK(!node->task_should_compute_output(i) ||
                    !accumulates_elsewhere(node->next_edge(i).function.get()),
                name, ": a backward pass is being captured while a graph of "
                "the same leaf that was made on another stream is alive; free "
                "that one first, or make it on the stream of the capture");
}

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// ------------------------------------------------------------- layer norm
struct LnShape {
  int64_t rows, width;
};

LnShape ln_shape(const Tensor& x) {
  const int64_t width = x.size(-1);
  return {x.numel() / width, width};
}

Tensor ln_forward(const Tensor& x, const Tensor& w, const Tensor& b,
                  const Tensor& res, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const auto [rows, width] = ln_shape(x);
  const Tensor& wide = res.defined() ? res : x;
  Tensor y = at::empty(x.sizes(), wide.options());
  if (stats)
    *stats = at::empty({3, rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return y;
  const Tensor xr = as_rows(x, rows, width);
  const Tensor rr = res.defined() ? as_rows(res, rows, width) : Tensor();
  const Tensor& affine = w.defined() ? w : b;
  check_launch(dear_ln_fwd(
      stream_of(x), type_code(x, "x"),
      res.defined() ? type_code(res, "residual") : -1,
      affine.defined() ? type_code(affine, "weight") : 0, data(xr),
      xr.stride(0), data(rr), res.defined() ? rr.stride(0) : 0, data(w),
      data(b), data(y), stats ? fdata(*stats) : nullptr, rows, (int)width,
      (float)eps));
  return y;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const Maybe& weight, const Maybe& bias,
                        const Maybe& residual, double eps) {
    const Tensor w = value(weight), b = value(bias), res = value(residual);
    Tensor stats;
    Tensor y = ln_forward(x, w, b, res, eps, &stats);
    // the bias itself is not needed, but its type is where there is no weight
    ctx->save_for_backward({x, w, res, stats, w.defined() ? Tensor() : b});
    ctx->saved_data["bias"] = b.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &res = saved[2],
                 &stats = saved[3];
    const Tensor& affine = w.defined() ? w : saved[4];
    const c10::DeviceGuard guard(x.device());
    check_operands({up[0]}, "layer_norm");
    check_capture(stream_of(x), "layer_norm");
    const auto [rows, width] = ln_shape(x);
    // the node has an edge for each tensor that was given
    const bool has_b = ctx->saved_data["bias"].toBool();
    size_t edge = 0;
    const bool want_x = ctx->needs_input_grad(edge++),
               want_w = w.defined() && ctx->needs_input_grad(edge++),
               want_b = has_b && ctx->needs_input_grad(edge++),
               want_r = res.defined() && ctx->needs_input_grad(edge++);
    // where the types are the same both sides of the sum share one gradient
    const bool same = want_x && want_r &&
                      x.scalar_type() == res.scalar_type();
    Tensor dx, dr, dw, db, part;
    if (want_x) dx = at::empty(x.sizes(), x.options());
    if (want_r && !same) dr = at::empty(res.sizes(), res.options());
    if (want_w) dw = at::empty({width}, affine.options());
    if (want_b) db = at::empty({width}, affine.options());
    if (rows == 0) {
      if (want_w) dw.zero_();
      if (want_b) db.zero_();
    } else {
      const Tensor xr = as_rows(x, rows, width);
      const Tensor rr = res.defined() ? as_rows(res, rows, width) : Tensor();
      const Tensor gr = as_rows(plain(up[0]), rows, width);
      const int64_t blocks = dear_ln_blocks(type_code(x, "x"), rows,
                                            (int)width);
      if (want_w || want_b)
        part = at::empty({blocks, 2, width}, stats.options());
      check_launch(dear_ln_bwd(
          stream_of(x), type_code(x, "x"),
          res.defined() ? type_code(res, "residual") : -1,
          affine.defined() ? type_code(affine, "weight") : 0, data(xr),
          xr.stride(0), data(rr), res.defined() ? rr.stride(0) : 0, data(gr),
          gr.stride(0), data(w), fdata(stats), data(dx), data(dr), data(dw),
          data(db), fdata(part), (int)blocks, rows, (int)width));
    }
    return once({dx, dw, db, same ? dx : dr, Tensor()}, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight,
                  const Maybe& bias, double eps,
                  const Maybe& residual) {
  Tensor a = plain(x), r = plain(value(residual));
  Tensor w = value(weight), b = value(bias);
  check_operands({a, r, w, b}, "layer_norm");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < kMaxWidth,
                    "layer_norm: x needs a last axis of 1 to 2^30 - 1 "
                    "elements");
  type_code(x, "layer_norm: x");
  if (r.defined()) {
    type_code(r, "layer_norm: residual");
    TORCH_CHECK_VALUE(r.sizes() == x.sizes() && r.device() == x.device(),
                      "layer_norm: the residual needs x's shape and device");
    // the sum is symmetric: the wider of two types is taken as the residual
    if (a.scalar_type() == at::kFloat && r.scalar_type() != at::kFloat)
      std::swap(a, r);
    TORCH_CHECK_TYPE(a.scalar_type() == r.scalar_type() ||
                         r.scalar_type() == at::kFloat,
                     "layer_norm: x and residual are of two 16-bit types");
  }
  const auto out = (r.defined() ? r : a).scalar_type();
  for (const Tensor* t : {&w, &b})
    if (t->defined()) {
      TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1) &&
                            t->device() == x.device() && t->is_contiguous(),
                        "layer_norm: weight and bias need shape (",
                        x.size(-1), ",), contiguous, on x's device");
      TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat ||
                           t->scalar_type() == out,
                       "layer_norm: weight and bias are float32 or of the "
                       "result's type");
    }
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() ||
                       w.scalar_type() == b.scalar_type(),
                   "layer_norm: weight and bias are of two types");
  TORCH_CHECK_VALUE(x.is_cuda(), "layer_norm: x is not on a GPU");
  w = plain(w);
  b = plain(b);
  if (!wants_grad({a, w, b, r})) return ln_forward(a, w, b, r, eps, nullptr);
  return LayerNormFn::apply(a, maybe(w), maybe(b), maybe(r), eps);
}

// ------------------------------------------------- token log probabilities
struct LogitRows {
  Tensor t;
  int64_t rows;
  int width;
};

LogitRows logit_rows(const Tensor& logits) {
  const int64_t width = logits.size(-1), rows = logits.numel() / width;
  return {rows ? as_rows(logits, rows, width) : logits, rows, (int)width};
}

void check_logits(const Tensor& t, const char* name) {
  type_code(t, "logits");
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1 &&
                        t.size(-1) < kMaxWidth,
                    name, ": logits need a last axis of 1 to 2^30 - 1 "
                    "tokens");
}

Tensor workspace(const Tensor& like, int64_t bytes) {
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// logprob (where there are tokens), entropy, and with top > 0 the top's log
// probabilities and ids
variable_list logprobs_forward(const Tensor& logits, const Tensor& tokens,
                               int64_t top, double t, int64_t ignore,
                               Tensor* stats) {
  const c10::DeviceGuard guard(logits.device());
  const auto z = logit_rows(logits);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const auto fopt = logits.options().dtype(at::kFloat);
  std::vector<int64_t> topped(lead.begin(), lead.end());
  topped.push_back(top);
  Tensor lp, h = at::empty(lead, fopt), tlp, tid;
  if (tokens.defined()) lp = at::empty(lead, fopt);
  if (top) {
    tlp = at::empty(topped, fopt);
    tid = at::empty(topped, logits.options().dtype(at::kLong));
  }
  if (stats) *stats = at::empty({z.rows, 4}, fopt);
  if (z.rows) {
    const Tensor tok = tokens.defined() ? tokens.contiguous() : Tensor();
    const int type = type_code(logits, "logits");
    const Tensor work = workspace(
        logits, dear_logprobs_work(type, z.rows, z.width, (int)top));
    check_launch(dear_logprobs_fwd(
        stream_of(logits), type, data(z.t),
        z.t.dim() == 2 ? z.t.stride(0) : 0, idata(tok), ignore, z.rows,
        z.width, (int)top, t, fdata(lp), fdata(h), fdata(tlp), idata(tid),
        stats ? data(*stats) : nullptr, data(work)));
  }
  variable_list out;
  if (tokens.defined()) out.push_back(lp);
  out.push_back(h);
  if (top) {
    out.push_back(tlp);
    out.push_back(tid);
  }
  return out;
}

Tensor up_of(const variable_list& up, size_t i) {
  return up[i].defined() ? plain(up[i]).contiguous() : Tensor();
}

struct LogprobsFn : torch::autograd::Function<LogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const Maybe& tokens_, int64_t top, double t,
                               int64_t ignore) {
    const Tensor tokens = value(tokens_);
    Tensor stats;
    auto out = logprobs_forward(logits, tokens, top, t, ignore, &stats);
    if (top) ctx->mark_non_differentiable({out.back()});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward(
        {logits, tokens, stats, top ? out.back() : Tensor()});
    ctx->saved_data["top"] = top;
    ctx->saved_data["t"] = t;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1];
    const c10::DeviceGuard guard(logits.device());
    for (const auto& u : up) check_operands({u}, "token_logprobs");
    check_capture(stream_of(logits), "token_logprobs");
    const int64_t top = ctx->saved_data["top"].toInt();
    const size_t at0 = tokens.defined() ? 1 : 0;
    const Tensor dlp = tokens.defined() ? up_of(up, 0) : Tensor();
    const Tensor dh = up_of(up, at0);
    const Tensor dtop = top ? up_of(up, at0 + 1) : Tensor();
    Tensor dz;
    if (dlp.defined() || dh.defined() || dtop.defined()) {
      dz = at::empty(logits.sizes(), logits.options());
      const auto z = logit_rows(logits);
      if (z.rows) {
        const Tensor tok = tokens.defined() ? tokens.contiguous() : Tensor();
        check_launch(dear_logprobs_bwd(
            stream_of(logits), type_code(logits, "logits"), data(z.t),
            z.t.dim() == 2 ? z.t.stride(0) : 0, idata(tok), idata(saved[3]),
            data(saved[2]), fdata(dlp), fdata(dh), fdata(dtop), data(dz),
            z.rows, z.width, (int)top, ctx->saved_data["t"].toDouble()));
      }
    }
    return once({dz, Tensor(), Tensor(), Tensor(), Tensor()},
                "token_logprobs");
  }
};

variable_list token_logprobs(const Tensor& logits_, const Maybe& tokens_,
                             int64_t top, double t, int64_t ignore) {
  const Tensor logits = plain(logits_), tokens = plain(value(tokens_));
  check_operands({logits, tokens}, "token_logprobs");
  check_logits(logits, "token_logprobs");
  TORCH_CHECK_VALUE(top >= 0 && top <= kMaxTop && top <= logits.size(-1),
                    "token_logprobs: top must be 0 to ", kMaxTop,
                    " and at most the vocabulary");
  if (tokens.defined())
    TORCH_CHECK_VALUE(
        tokens.scalar_type() == at::kLong &&
            tokens.device() == logits.device() &&
            tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
        "token_logprobs: tokens are int64, on the logits' device, one for "
        "each row");
  TORCH_CHECK_VALUE(logits.is_cuda(),
                    "token_logprobs: logits are not on a GPU");
  if (!wants_grad({logits}))
    return logprobs_forward(logits, tokens, top, t, ignore, nullptr);
  return LogprobsFn::apply(logits, maybe(tokens), top, t, ignore);
}

// ------------------------------------------------------------ distillation
// `kept`: for the backward pass, four numbers a row, and behind them the named
// tokens' gradients
Tensor distill_forward(const Tensor& logits, const Tensor& ids,
                       const Tensor& teacher, double t, bool tail,
                       Tensor* kept) {
  const c10::DeviceGuard guard(logits.device());
  const auto z = logit_rows(logits);
  const auto fopt = logits.options().dtype(at::kFloat);
  const int64_t k = ids.size(-1);
  Tensor loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), fopt);
  if (kept) *kept = at::empty({z.rows * (4 + k)}, fopt);
  if (z.rows) {
    const Tensor idc = ids.contiguous();
    const Tensor tc = teacher.to(at::kFloat).contiguous();
    const int type = type_code(logits, "logits");
    const Tensor work = workspace(
        logits, dear_distill_work(type, z.rows, z.width));
    float* stats = kept ? fdata(*kept) : nullptr;
    check_launch(dear_distill_fwd(
        stream_of(logits), type, tail, data(z.t),
        z.t.dim() == 2 ? z.t.stride(0) : 0, idata(idc), fdata(tc), z.rows,
        z.width, (int)k, t, fdata(loss),
        stats ? stats + z.rows * 4 : nullptr, stats, data(work)));
  }
  return loss;
}

struct DistillFn : torch::autograd::Function<DistillFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits,
                        const Tensor& ids, const Tensor& teacher, double t,
                        bool tail) {
    Tensor kept;
    Tensor loss = distill_forward(logits, ids, teacher, t, tail, &kept);
    ctx->save_for_backward({logits, ids, kept});
    ctx->saved_data["t"] = t;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &ids = saved[1];
    const c10::DeviceGuard guard(logits.device());
    check_operands({up[0]}, "topk_distill_loss");
    check_capture(stream_of(logits), "topk_distill_loss");
    const auto z = logit_rows(logits);
    Tensor dz = at::empty(logits.sizes(), logits.options());
    if (z.rows) {
      const Tensor idc = ids.contiguous(), g = up_of(up, 0);
      check_launch(dear_distill_bwd(
          stream_of(logits), type_code(logits, "logits"), data(z.t),
          z.t.dim() == 2 ? z.t.stride(0) : 0, idata(idc),
          fdata(saved[2]) + z.rows * 4, data(saved[2]), fdata(g), data(dz),
          z.rows, z.width,
          (int)ids.size(-1), ctx->saved_data["t"].toDouble()));
    }
    return once({dz, Tensor(), Tensor(), Tensor(), Tensor()},
                "topk_distill_loss");
  }
};

Tensor topk_distill_loss(const Tensor& logits_, const Tensor& ids_,
                         const Tensor& teacher_, double t, bool tail) {
  const Tensor logits = plain(logits_), ids = plain(ids_),
               teacher = plain(teacher_);
  check_operands({logits, ids, teacher}, "topk_distill_loss");
  check_logits(logits, "topk_distill_loss");
  type_code(teacher, "top_logprobs");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(
      ids.scalar_type() == at::kLong && ids.device() == logits.device() &&
          teacher.device() == logits.device() &&
          ids.sizes() == teacher.sizes() && ids.dim() == logits.dim() &&
          ids.sizes().slice(0, ids.dim() - 1) == lead,
      "topk_distill_loss: top_ids (int64) and top_logprobs have the logits' "
      "leading shape and device, and one length");
  TORCH_CHECK_VALUE(ids.size(-1) >= 1 && ids.size(-1) <= kMaxTop,
                    "topk_distill_loss: 1 to ", kMaxTop, " entries a row");
  TORCH_CHECK_VALUE(logits.is_cuda(),
                    "topk_distill_loss: logits are not on a GPU");
  if (!wants_grad({logits}))
    return distill_forward(logits, ids, teacher, t, tail, nullptr);
  return DistillFn::apply(logits, ids, teacher, t, tail);
}

}  // namespace

void register_lm_ops(pybind11::module& m) {
  namespace py = pybind11;
  const auto free = py::call_guard<py::gil_scoped_release>();
  m.attr("max_top") = kMaxTop;
  m.def("layer_norm", &layer_norm, free);
  m.def("token_logprobs", &token_logprobs, free);
  m.def("topk_distill_loss", &topk_distill_loss, free);
}
