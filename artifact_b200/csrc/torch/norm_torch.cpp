// The torch side of layer norm and dropout: argument checks, memory, and autograd nodes over the C ABI of
// include/rof_b200.h.  In C++ because the operators are short: between two layers of a small graph a training step of
// one of them is 10 us of kernels, and an autograd node written in Python costs 60 us more than one that is not.
//
// artifact_b200/norm.py documents the operators and hands their arguments through.
#include <ATen/TracerMode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/types.h>

#include <optional>
#include <tuple>
#include <vector>

#include "rof_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

int dtype_code(at::ScalarType t) { return t == at::kFloat ? ROF_DTYPE_F32 : t == at::kBFloat16 ? ROF_DTYPE_BF16 : ROF_DTYPE_F16; }

// What the operators do not offer is refused: without a node of its own the result would carry no tangent, and a trace records the
// allocation of the result alone.
void check_call(const char* who, const Tensor& x, const MaybeTensor& a, const MaybeTensor& b) {
  const auto dual = [](const Tensor& t) { return t._fw_grad(0).defined(); };
  TORCH_CHECK(!dual(x) && !(a.has_value() && dual(*a)) && !(b.has_value() && dual(*b)), who, " has no forward-mode derivative");
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(), who, " cannot be traced (torch.jit.trace)");
}

void check_matrix(const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const at::ScalarType t = x.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "x must be float32, bfloat16 or float16, got ", t);
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
}

void check_vector(const MaybeTensor& v, const char* name, const Tensor& x) {
  if (!v.has_value()) return;
  TORCH_CHECK(v->device() == x.device() && v->dim() == 1 && v->size(0) == x.size(-1), name, " must be a vector of ", x.size(-1),
              " entries on x's device, got ", v->sizes(), " on ", v->device());
  TORCH_CHECK(v->scalar_type() == at::kFloat || v->scalar_type() == x.scalar_type(), name, " must be float32 or of x's type, got ",
              v->scalar_type());
}

// a dropout (p = 0: none); a 64-bit word per number, as the autograd node keeps them
struct Drop {
  double p;
  int64_t seed, step, first_row;
  rof_dropout c(const Tensor& step_tensor) const {
    return rof_dropout{p, (uint64_t)seed, (uint64_t)step, step_tensor.defined() ? step_tensor.const_data_ptr<int64_t>() : nullptr, first_row};
  }
};

void check_drop(const Drop& d, const MaybeTensor& step, const Tensor& x) {
  TORCH_CHECK_VALUE(d.p >= 0.0 && d.p <= 1.0, "p must be in [0, 1], got ", d.p);
  TORCH_CHECK_VALUE(d.first_row >= 0, "row_offset must not be negative, got ", d.first_row);
  TORCH_CHECK(!step.has_value() || (step->scalar_type() == at::kLong && step->numel() == 1 && step->device() == x.device() && !step->is_neg()),
              "step must be a number or a one-element int64 tensor on x's device");
}

void check_status(int status) {
  TORCH_CHECK(status == ROF_OK, "rof_b200 status ", status, ": ", rof_last_error());
}

// a lazily negated view's memory holds the negatives of its values (the question first: the call costs a microsecond)
Tensor resolved(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// x as [rows, width] with unit column stride: a view where its layout allows it, else a copy
Tensor rows_of(const Tensor& given) {
  const Tensor x = resolved(given);
  const Tensor v = x.dim() == 2 ? x : x.dim() == 1 ? x.unsqueeze(0) : x.flatten(0, -2);
  if (v.is_contiguous() || ((v.stride(1) == 1 || v.size(1) <= 1) && (v.stride(0) >= v.size(1) || v.size(0) <= 1))) return v;
  return v.contiguous();
}

int64_t offset_of(const Tensor& t) { return (int64_t)(reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16); }

// t with rows that lie against the 16-byte boundaries like v's: t itself, or a copy.  The backward kernels read both
// matrices in the same 16-byte vectors; a copy costs a third of what they lose on rows that lie differently.
Tensor laid_like(const Tensor& t, const Tensor& v) {
  const int64_t per = 16 / t.element_size(), step = v.stride(0) % per;
  if (offset_of(t) == offset_of(v) && (t.stride(0) % per == step || t.size(0) <= 1)) return t;
  const int64_t rows = t.size(0), width = t.size(1), lead = ((rows > 1 ? step : 0) - width % per + per) % per;
  const Tensor flat = at::empty({rows * (width + lead) + per}, t.options());
  Tensor out = flat.as_strided({rows, width}, {width + lead, 1}, offset_of(v) / t.element_size());
  out.copy_(t);
  return out;
}

Tensor empty_like_rows(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

// the one type in which both vectors go down: their own, or 32-bit where they differ
at::ScalarType kind_of(const Tensor& weight, const Tensor& bias) {
  if (!weight.defined() || !bias.defined()) {
    const Tensor& v = weight.defined() ? weight : bias;
    return v.defined() ? v.scalar_type() : at::kFloat;
  }
  return weight.scalar_type() == bias.scalar_type() ? weight.scalar_type() : at::kFloat;
}

Tensor vector_of(const Tensor& v, at::ScalarType kind) { return v.defined() ? resolved(v.scalar_type() == kind ? v : v.to(kind)).contiguous() : v; }

const void* pointer(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_pointer(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& x) { return at::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

Tensor workspace_of(int64_t rows, int64_t width, const Tensor& x) {
  // torch's caching allocator returns 512-byte aligned blocks
  return at::empty({rof_layer_norm_workspace_bytes(rows, (int)width)}, x.options().dtype(at::kByte));
}

int width_of(const Tensor& v) {
  TORCH_CHECK(v.size(1) <= (1 << 30), "rows of more than 2^30 columns");
  return (int)v.size(1);
}

// ---- layer norm ---------------------------------------------------------------------------------
// -> x as rows, y, the rows' statistics (undefined where not wanted)
std::tuple<Tensor, Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool relu,
                                                const Drop& drop, const Tensor& step, bool want_stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor v = rows_of(x), y = empty_like_rows(x);
  const int width = width_of(v);
  const Tensor stats = want_stats ? at::empty({v.size(0), 2}, x.options().dtype(at::kFloat)) : Tensor();
  const at::ScalarType kind = kind_of(weight, bias);
  const Tensor w = vector_of(weight, kind), b = vector_of(bias, kind);
  const rof_dropout d = drop.c(step);
  check_status(rof_layer_norm_forward(dtype_code(x.scalar_type()), v.const_data_ptr(), v.stride(0), v.size(0), width, dtype_code(kind),
                                      pointer(w), pointer(b), (float)eps, relu, drop.p > 0.0 ? &d : nullptr, y.mutable_data_ptr(), width,
                                      static_cast<float*>(mutable_pointer(stats)), stream_of(x)));
  return {v, y, stats};
}

// Gradients that refuse to be differentiated again, where a graph of them is being made (create_graph).
variable_list once(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string(who) + " has no second derivative", (int64_t)grads.size());
  variable_list inputs;
  for (const Tensor& g : grads) inputs.push_back(g.defined() ? g.detach().requires_grad_(g.is_floating_point()) : g);
  return (*error)(std::move(inputs));
}

// What a backward pass gets back of what was saved.  Hooks on saved tensors may hand back something else, which the kernels must not
// read: they get pointers.
void check_saved(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef sizes, const Tensor& dy) {
  TORCH_CHECK(t.defined() && t.device() == dy.device() && t.scalar_type() == type && t.sizes() == sizes, "a hook on saved tensors returned ",
              t.defined() ? t.sizes() : at::IntArrayRef(), " ", t.defined() ? c10::toString(t.scalar_type()) : "nothing", " for ", name,
              ", not what was saved");
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, bool relu,
                        double p, int64_t seed, int64_t step, int64_t first_row, const MaybeTensor& step_tensor) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor()), t = step_tensor.value_or(Tensor());
    auto [v, y, stats] = norm_forward(x, w, b, eps, relu, Drop{p, seed, step, first_row}, t, true);
    ctx->save_for_backward({v, w, b, stats, t});
    ctx->saved_data["drop"] = std::vector<int64_t>{seed, step, first_row, relu};
    ctx->saved_data["p"] = p;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &weight = saved[1], &bias = saved[2];
    const auto numbers = ctx->saved_data["drop"].toIntVector();
    const Drop drop{ctx->saved_data["p"].toDouble(), numbers[0], numbers[1], numbers[2]};
    variable_list out(10);
    if (!grads[0].defined()) return out;
    // (the node counts the tensors it was given, not the places of arguments)
    const bool need_x = ctx->needs_input_grad(0), need_w = weight.defined() && ctx->needs_input_grad(1),
               need_b = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(grads[0].device());
      const Tensor g = rows_of(grads[0]);
      const int64_t rows = g.size(0);
      const int width = (int)g.size(1);
      check_saved(saved[0], "x", g.scalar_type(), {rows, width}, g);
      check_saved(saved[3], "the rows' statistics", at::kFloat, {rows, 2}, g);
      check_vector(weight.defined() ? MaybeTensor(weight) : std::nullopt, "weight", g);
      check_vector(bias.defined() ? MaybeTensor(bias) : std::nullopt, "bias", g);
      check_drop(drop, saved[4].defined() ? MaybeTensor(saved[4]) : std::nullopt, g);
      const Tensor v = rows_of(saved[0]), stats = saved[3].contiguous(), dy = laid_like(g, v);
      const at::ScalarType kind = kind_of(weight, bias);
      const Tensor w = vector_of(weight, kind), b = vector_of(bias, kind);
      Tensor dx, dw, db, ws;
      if (need_x) dx = empty_like_rows(grads[0]);
      if (need_w) dw = at::empty({width}, w.options());
      if (need_b) db = at::empty({width}, b.options());
      if (need_w || need_b) ws = workspace_of(rows, width, v);
      const rof_dropout d = drop.c(saved[4]);
      check_status(rof_layer_norm_backward(dtype_code(v.scalar_type()), dy.const_data_ptr(), dy.stride(0), v.const_data_ptr(), v.stride(0), rows,
                                           width, dtype_code(kind), pointer(w), pointer(b), static_cast<const float*>(stats.const_data_ptr()),
                                           (int)numbers[3], drop.p > 0.0 ? &d : nullptr, mutable_pointer(dx), width, mutable_pointer(dw),
                                           mutable_pointer(db), mutable_pointer(ws), ws.defined() ? ws.numel() : 0, stream_of(v)));
      out[0] = dx;
      if (need_w) out[1] = dw.to(weight.scalar_type());
      if (need_b) out[2] = db.to(bias.scalar_type());
    }
    return once(std::move(out), "layer_norm");
  }
};

bool needs_graph(const Tensor& x, const MaybeTensor& a, const MaybeTensor& b) {
  return at::GradMode::is_enabled() && (x.requires_grad() || (a.has_value() && a->requires_grad()) || (b.has_value() && b->requires_grad()));
}

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps, bool relu, double p, uint64_t seed,
                  uint64_t step, int64_t first_row, const MaybeTensor& step_tensor) {
  check_call("layer_norm", x, weight, bias);
  check_matrix(x);
  check_vector(weight, "weight", x);
  check_vector(bias, "bias", x);
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got ", eps);
  const Drop drop{p, (int64_t)seed, (int64_t)step, first_row};
  check_drop(drop, step_tensor, x);
  if (needs_graph(x, weight, bias))
    return LayerNorm::apply(x, weight, bias, eps, relu, p, drop.seed, drop.step, first_row, step_tensor);
  return std::get<1>(norm_forward(x, weight.value_or(Tensor()), bias.value_or(Tensor()), eps, relu, drop, step_tensor.value_or(Tensor()), false));
}

// ---- dropout ------------------------------------------------------------------------------------
Tensor dropout_forward(const Tensor& x, const Tensor& bias, bool relu, const Drop& drop, const Tensor& step) {
  const c10::DeviceGuard guard(x.device());
  const Tensor v = rows_of(x), y = empty_like_rows(x);
  const int width = width_of(v);
  const Tensor b = bias.defined() ? vector_of(bias, bias.scalar_type()) : bias;
  const rof_dropout d = drop.c(step);
  check_status(rof_dropout_forward(dtype_code(x.scalar_type()), v.const_data_ptr(), v.stride(0), v.size(0), width,
                                   dtype_code(b.defined() ? b.scalar_type() : at::kFloat), pointer(b), relu, drop.p > 0.0 ? &d : nullptr,
                                   y.mutable_data_ptr(), width, stream_of(x)));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& bias, bool relu, double p, int64_t seed, int64_t step,
                        int64_t first_row, const MaybeTensor& step_tensor) {
    const Tensor t = step_tensor.value_or(Tensor());
    const Tensor y = dropout_forward(x, bias.value_or(Tensor()), relu, Drop{p, seed, step, first_row}, t);
    // behind a ReLU the output's bits say which elements were kept and positive
    ctx->save_for_backward({relu ? y : Tensor(), t});
    ctx->saved_data["drop"] = std::vector<int64_t>{seed, step, first_row, relu, bias.has_value(),
                                                   bias.has_value() && bias->scalar_type() == at::kFloat};
    ctx->saved_data["p"] = p;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& y = saved[0];
    const auto numbers = ctx->saved_data["drop"].toIntVector();
    const Drop drop{ctx->saved_data["p"].toDouble(), numbers[0], numbers[1], numbers[2]};
    variable_list out(8);
    if (!grads[0].defined()) return out;
    const bool need_x = ctx->needs_input_grad(0), need_b = numbers[4] && ctx->needs_input_grad(1);
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(grads[0].device());
      Tensor dy = rows_of(grads[0]);
      const int64_t rows = dy.size(0);
      const int width = (int)dy.size(1);
      if (numbers[3]) check_saved(y, "the output", dy.scalar_type(), grads[0].sizes(), dy);
      check_drop(drop, saved[1].defined() ? MaybeTensor(saved[1]) : std::nullopt, dy);
      const Tensor yy = y.defined() ? rows_of(y) : y;
      const at::ScalarType kind = numbers[5] ? at::kFloat : dy.scalar_type();
      Tensor dx, db, ws;
      if (need_x) dx = empty_like_rows(grads[0]);
      if (need_b) {
        if (need_x || y.defined()) dy = laid_like(dy, need_x ? rows_of(dx) : yy);
        db = at::empty({width}, dy.options().dtype(kind));
        ws = workspace_of(rows, width, dy);
      }
      const rof_dropout d = drop.c(saved[1]);
      check_status(rof_dropout_backward(dtype_code(dy.scalar_type()), dy.const_data_ptr(), dy.stride(0), pointer(yy), yy.defined() ? yy.stride(0) : width, rows, width,
                                        dtype_code(kind), (int)numbers[3], drop.p > 0.0 ? &d : nullptr, mutable_pointer(dx), width,
                                        mutable_pointer(db), mutable_pointer(ws), ws.defined() ? ws.numel() : 0, stream_of(dy)));
      out[0] = dx;
      out[1] = db;
    }
    return once(std::move(out), "dropout");
  }
};

Tensor dropout(const Tensor& x, const MaybeTensor& bias, bool relu, double p, uint64_t seed, uint64_t step, int64_t first_row,
               const MaybeTensor& step_tensor) {
  check_call("dropout", x, bias, std::nullopt);
  check_matrix(x);
  check_vector(bias, "bias", x);
  const Drop drop{p, (int64_t)seed, (int64_t)step, first_row};
  check_drop(drop, step_tensor, x);
  if (needs_graph(x, bias, std::nullopt)) return Dropout::apply(x, bias, relu, p, drop.seed, drop.step, first_row, step_tensor);
  return dropout_forward(x, bias.value_or(Tensor()), relu, drop, step_tensor.value_or(Tensor()));
}

}  // namespace

PYBIND11_MODULE(rof_torch, m) {
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layer_norm", &layer_norm, free);
  m.def("dropout", &dropout, free);
  m.def("rows_of", &rows_of, free);
  m.def("laid_like", &laid_like, free);
}
