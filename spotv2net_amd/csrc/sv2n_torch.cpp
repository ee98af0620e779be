// The layer-norm operators' host side in C++: their kernels take a few microseconds,
// less than an operator implemented in Python costs to call, and an autograd node in
// Python costs more than both passes.  Registers, for the schemas library.py defines,
//   sv2n::layer_norm          CUDA kernel and autograd formula
//   sv2n::layer_norm_bwd      CUDA kernel; not differentiable, which it says
//   sv2n::layer_norm_bwd_acc  CUDA kernel
// The C entries come from whichever libsv2n build the process loaded: _lib.py hands
// their addresses to sv2n_torch_bind before the first call.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "sv2n.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&sv2n_layer_norm_fwd) fwd = nullptr;
  decltype(&sv2n_layer_norm_bwd) bwd = nullptr;
  decltype(&sv2n_layer_norm_bwd_workspace) bwd_ws = nullptr;
  decltype(&sv2n_strerror) strerror = nullptr;
} g_entries;

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", g_entries.strerror(rc));
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SV2N_DT_F32;
    case at::kBFloat16: return SV2N_DT_BF16;
    case at::kHalf: return SV2N_DT_F16;
    default: return -1;
  }
}

// x as [rows, cols] with unit column stride and a row stride of at least a row: a view
// where its strides allow one, else a dense copy
Tensor rows_of(const Tensor& x) {
  const int64_t cols = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, cols});
  if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < cols)) r = r.contiguous();
  return r;
}
int64_t row_stride(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

// Refuses what the kernels do not take; the type code of the weight
int check_inputs(const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  TORCH_CHECK(g_entries.fwd, "sv2n: the kernels' library is not loaded");
  TORCH_CHECK(x.dim() >= 1, "sv2n: layer_norm: expected at least one dimension");
  const int64_t cols = x.size(-1);
  TORCH_CHECK(dtype_code(x.scalar_type()) >= 0,
              "sv2n: layer_norm: expected float32, bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK(cols >= 1 && cols <= SV2N_LN_MAX_COLS, "sv2n: layer_norm: rows of 1 to ",
              SV2N_LN_MAX_COLS, " elements, got ", cols);
  std::optional<at::ScalarType> type;
  const char* name = "weight";
  for (const OptTensor* t : {&weight, &bias}) {
    if (t->has_value()) {
      const Tensor& v = **t;
      TORCH_CHECK(v.dim() == 1 && v.size(0) == cols, "sv2n: layer_norm: ", name, " of shape ",
                  v.sizes(), " for rows of ", cols);
      TORCH_CHECK(v.device() == x.device(), "sv2n: layer_norm: ", name, " on ", v.device(),
                  ", input on ", x.device());
      TORCH_CHECK(v.scalar_type() == at::kFloat || v.scalar_type() == x.scalar_type(),
                  "sv2n: layer_norm: ", name, " is ", v.scalar_type(),
                  "; expected float32 or the input's ", x.scalar_type());
      TORCH_CHECK(!type || *type == v.scalar_type(),
                  "sv2n: layer_norm: weight and bias of different types");
      type = v.scalar_type();
    }
    name = "bias";
  }
  return dtype_code(type.value_or(x.scalar_type()));
}

hipStream_t stream_of(const Tensor& x) {
  return c10::hip::getCurrentHIPStream(x.device().index()).stream();
}

const void* data_of(const Tensor& t) { return t.numel() ? t.const_data_ptr() : nullptr; }

std::tuple<Tensor, Tensor, Tensor> layer_norm(const Tensor& x, const OptTensor& weight,
                                              const OptTensor& bias, double eps) {
  const int wdt = check_inputs(x, weight, bias);
  TORCH_CHECK(eps >= 0.0, "sv2n: layer_norm: eps must not be negative, got ", eps);
  const c10::OptionalDeviceGuard guard(x.device());
  const Tensor r = rows_of(x);
  const int64_t rows = r.size(0), cols = r.size(1);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor mean = at::empty({rows}, x.options().dtype(at::kFloat));
  Tensor rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (rows) {
    const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
    check(g_entries.fwd(r.const_data_ptr(), row_stride(r), dtype_code(x.scalar_type()),
                        w.defined() ? w.const_data_ptr() : nullptr,
                        b.defined() ? b.const_data_ptr() : nullptr, wdt, rows, (int)cols, (float)eps,
                        y.mutable_data_ptr(), mean.mutable_data_ptr<float>(),
                        rstd.mutable_data_ptr<float>(), stream_of(x)),
          "sv2n_layer_norm_fwd");
  }
  return {y, mean, rstd};
}

// dx (undefined unless asked for); dw and db into what is given
Tensor backward_into(const Tensor& dy, const Tensor& x, const OptTensor& weight, const Tensor& mean,
                     const Tensor& rstd, bool need_dx, const OptTensor& dw, const OptTensor& db,
                     bool accumulate) {
  int wdt = check_inputs(x, weight, std::nullopt);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() &&
                  dy.device() == x.device(),
              "sv2n: layer_norm_bwd: dy ", dy.sizes(), " ", dy.scalar_type(), " for x ", x.sizes(),
              " ", x.scalar_type());
  const c10::OptionalDeviceGuard guard(x.device());
  const Tensor r = rows_of(x), d = rows_of(dy);
  const int64_t rows = r.size(0), cols = r.size(1);
  for (const Tensor* t : {&mean, &rstd})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->numel() == rows && t->is_contiguous() &&
                    t->device() == x.device(),
                "sv2n: layer_norm_bwd: mean / rstd are the forward's");
  for (const OptTensor* g : {&dw, &db}) {
    if (!g->has_value()) continue;
    const Tensor& v = **g;
    TORCH_CHECK(v.dim() == 1 && v.size(0) == cols && v.is_contiguous() && v.device() == x.device() &&
                    (v.scalar_type() == at::kFloat || v.scalar_type() == x.scalar_type()),
                "sv2n: layer_norm_bwd: gradient buffer");
    if (!weight) wdt = dtype_code(v.scalar_type());
    TORCH_CHECK(dtype_code(v.scalar_type()) == wdt,
                "sv2n: layer_norm_bwd: gradients and weight of different types");
  }
  if (dw && db) {
    const auto a = (uintptr_t)dw->const_data_ptr(), b = (uintptr_t)db->const_data_ptr();
    const uintptr_t n = cols * dw->element_size();
    TORCH_CHECK(a + n <= b || b + n <= a, "sv2n: layer_norm_bwd: the gradient buffers overlap");
  }
  Tensor dx;
  if (need_dx) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  const bool wg = dw.has_value() || db.has_value();
  const int dt = dtype_code(x.scalar_type());
  const int64_t ws_n = wg ? g_entries.bwd_ws(rows, (int)cols, dt) : 0;
  Tensor ws;
  if (ws_n) ws = at::empty({ws_n}, x.options().dtype(at::kFloat));
  const Tensor w = weight ? weight->contiguous() : Tensor();
  check(g_entries.bwd(data_of(d), row_stride(d), data_of(r), row_stride(r), dt,
                      w.defined() ? w.const_data_ptr() : nullptr, wdt,
                      (const float*)data_of(mean), (const float*)data_of(rstd), rows, (int)cols,
                      dx.defined() && dx.numel() ? dx.mutable_data_ptr() : nullptr,
                      dw ? dw->mutable_data_ptr() : nullptr, db ? db->mutable_data_ptr() : nullptr,
                      accumulate, ws_n ? ws.mutable_data_ptr<float>() : nullptr, ws_n,
                      stream_of(x)),
        "sv2n_layer_norm_bwd");
  return dx;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& dy, const Tensor& x,
                                                  const OptTensor& weight, const Tensor& mean,
                                                  const Tensor& rstd, bool need_dx, bool need_dw,
                                                  bool need_db,
                                                  std::optional<at::ScalarType> grad_dtype) {
  const auto type = weight ? weight->scalar_type() : grad_dtype.value_or(x.scalar_type());
  const auto opts = x.options().dtype(type);
  const int64_t cols = x.dim() ? x.size(-1) : 0;
  OptTensor dw, db;
  if (need_dw) dw = at::empty({cols}, opts);
  if (need_db) db = at::empty({cols}, opts);
  Tensor dx = backward_into(dy, x, weight, mean, rstd, need_dx, dw, db, false);
  auto or_none = [&](const Tensor& t) { return t.defined() ? t : at::empty({0}, x.options()); };
  return {or_none(dx), or_none(dw.value_or(Tensor())), or_none(db.value_or(Tensor()))};
}

Tensor layer_norm_bwd_acc(const Tensor& dy, const Tensor& x, const OptTensor& weight,
                          const Tensor& mean, const Tensor& rstd, const OptTensor& g_weight,
                          const OptTensor& g_bias) {
  return backward_into(dy, x, weight, mean, rstd, true, g_weight, g_bias, true);
}

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

std::tuple<Tensor, Tensor, Tensor> call_layer_norm(const Tensor& x, const OptTensor& weight,
                                                   const OptTensor& bias, double eps) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("sv2n::layer_norm", "")
                       .typed<decltype(layer_norm)>();
  return op.call(x, weight, bias, eps);
}
std::tuple<Tensor, Tensor, Tensor> call_layer_norm_bwd(const Tensor& dy, const Tensor& x,
                                                       const OptTensor& weight, const Tensor& mean,
                                                       const Tensor& rstd, bool need_dx,
                                                       bool need_dw, bool need_db,
                                                       std::optional<at::ScalarType> grad_dtype) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("sv2n::layer_norm_bwd", "")
                       .typed<decltype(layer_norm_bwd)>();
  return op.call(dy, x, weight, mean, rstd, need_dx, need_dw, need_db, grad_dtype);
}

// The backward's node.  (A Node of its own rather than a custom Function: the wrapping a
// Function does around both passes costs more than the kernels of a small call.)
struct LayerNormBackward : torch::autograd::Node {
  SavedVariable x, weight, mean, rstd;
  bool has_weight = false, has_bias = false;
  at::ScalarType bias_type = at::kFloat;
  bool released = false;

  std::string name() const override { return "LayerNormBackward"; }

  // A leaf's accumulation node lives as long as any graph of the leaf and keeps the
  // stream it was made on.  If that is the default stream, the engine would make it wait
  // for a stream that is being captured, which ends the process; here it is an error.
  void refuse_capture_from_eager() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (uint32_t i = 0; i < num_outputs(); ++i) {
      const auto& next = next_edge(i).function;
      if (!task_should_compute_output(i) ||
          !dynamic_cast<torch::autograd::AccumulateGrad*>(next.get()))
        continue;
      const auto s = next->stream();
      TORCH_CHECK(!s || s->id() != c10::hip::getDefaultHIPStream(s->device_index()).id(),
                  "sv2n: layer_norm's backward is being captured while an eager graph of the "
                  "same leaf, built on the default stream, is alive: delete it first");
    }
  }

  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
    refuse_capture_from_eager();
    // (unpacking may run a checkpointed forward again, and the call is itself recorded
    // where gradients of the gradients are: neither below autograd)
    const Tensor xv = x.unpack(), mv = mean.unpack(), rv = rstd.unpack();
    const OptTensor w = has_weight ? OptTensor(weight.unpack()) : std::nullopt;
    const bool nx = task_should_compute_output(0);
    const bool nw = has_weight && task_should_compute_output(1);
    const bool nb = has_bias && task_should_compute_output(2);
    auto [dx, dw, db] = call_layer_norm_bwd(
        grads[0], xv, w, mv, rv, nx, nw, nb,
        has_bias ? std::optional<at::ScalarType>(bias_type) : std::nullopt);
    if (nx) out[0] = std::move(dx);
    if (nw) out[1] = std::move(dw);
    if (nb) out[2] = std::move(db);
    return out;
  }
  void release_variables() override {
    released = true;
    for (SavedVariable* v : {&x, &weight, &mean, &rstd}) v->reset_data();
  }
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_autograd(const Tensor& x, const OptTensor& weight,
                                                       const OptTensor& bias, double eps) {
  const bool need = at::GradMode::is_enabled() &&
                    (x.requires_grad() || (weight && weight->requires_grad()) ||
                     (bias && bias->requires_grad()));
  for (const OptTensor& t : {OptTensor(x), weight, bias})
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t),
                "sv2n: layer_norm has no forward-mode derivative");
  std::tuple<Tensor, Tensor, Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = call_layer_norm(x, weight, bias, eps);
  }
  if (!need) return out;
  std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
  node->x = SavedVariable(x, false);
  node->has_weight = w.defined();
  if (node->has_weight) node->weight = SavedVariable(w, false);
  node->has_bias = b.defined();
  if (node->has_bias) node->bias_type = b.scalar_type();
  node->mean = SavedVariable(std::get<1>(out), false);
  node->rstd = SavedVariable(std::get<2>(out), false);
  torch::autograd::set_history(std::get<0>(out), node);
  return out;
}

// What the gradients depend on, for whoever differentiates them: an error
struct LayerNormOnce : torch::autograd::Node {
  std::string name() const override { return "LayerNormOnce"; }
  variable_list apply(variable_list&&) override {
    TORCH_CHECK(false, "sv2n: layer_norm is differentiable once (its gradients have no gradient)");
  }
};

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd_autograd(
    const Tensor& dy, const Tensor& x, const OptTensor& weight, const Tensor& mean,
    const Tensor& rstd, bool need_dx, bool need_dw, bool need_db,
    std::optional<at::ScalarType> grad_dtype) {
  const Tensor w = weight.value_or(Tensor());
  for (const OptTensor& t : {OptTensor(dy), OptTensor(x), weight})
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t),
                "sv2n: layer_norm is differentiable once (its gradients have no gradient)");
  std::tuple<Tensor, Tensor, Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = call_layer_norm_bwd(dy, x, weight, mean, rstd, need_dx, need_dw, need_db, grad_dtype);
  }
  if (at::GradMode::is_enabled() &&
      (dy.requires_grad() || x.requires_grad() || (w.defined() && w.requires_grad()) ||
       mean.requires_grad() || rstd.requires_grad())) {
    std::shared_ptr<LayerNormOnce> node(new LayerNormOnce(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(dy, x, w, mean, rstd));
    if (need_dx) torch::autograd::set_history(std::get<0>(out), node);
    if (need_dw) torch::autograd::set_history(std::get<1>(out), node);
    if (need_db) torch::autograd::set_history(std::get<2>(out), node);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(sv2n, CUDA, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("layer_norm_bwd", layer_norm_bwd);
  m.impl("layer_norm_bwd_acc", layer_norm_bwd_acc);
}
TORCH_LIBRARY_IMPL(sv2n, Autograd, m) {
  m.impl("layer_norm", layer_norm_autograd);
  m.impl("layer_norm_bwd", layer_norm_bwd_autograd);
}

extern "C" void sv2n_torch_bind(void* fwd, void* bwd, void* bwd_ws, void* strerror) {
  g_entries.fwd = (decltype(g_entries.fwd))fwd;
  g_entries.bwd = (decltype(g_entries.bwd))bwd;
  g_entries.bwd_ws = (decltype(g_entries.bwd_ws))bwd_ws;
  g_entries.strerror = (decltype(g_entries.strerror))strerror;
}
