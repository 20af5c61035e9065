// torch binding of the decoder losses (clip_linear_ce / clip_linear_distill / clip_topk_scores of include/clip_amd.h):
// argument checks, output and workspace tensors, and the autograd node, in C++.  At a few dozen rows a training step is
// host time: torch runs a backward pass on a thread of its own, where a Python node pays for the interpreter lock and cold
// caches on every line (forward + backward of 37 rows: 215 us through a Python autograd.Function and ctypes).
// Nothing is computed here, and there is no fallback: every call goes to libclip_amd.so, whose entry points the Python host
// hands over (so that CLIP_AMD_LIB holds for both).
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include "../../include/clip_amd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::isFwGradDefined;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct Entry {
  decltype(&clip_linear_loss_workspace) workspace;
  decltype(&clip_linear_ce) ce;
  decltype(&clip_linear_ce_grad) ce_grad;
  decltype(&clip_linear_distill) distill;
  decltype(&clip_linear_distill_grad) distill_grad;
  decltype(&clip_topk_scores) topk;
  decltype(&clip_last_error) last_error;
} entry;

void bind(const std::vector<uintptr_t>& p) {
  TORCH_CHECK(p.size() == 7, "bind: seven entry points");
  entry = Entry{reinterpret_cast<decltype(Entry::workspace)>(p[0]), reinterpret_cast<decltype(Entry::ce)>(p[1]),
                reinterpret_cast<decltype(Entry::ce_grad)>(p[2]),   reinterpret_cast<decltype(Entry::distill)>(p[3]),
                reinterpret_cast<decltype(Entry::distill_grad)>(p[4]), reinterpret_cast<decltype(Entry::topk)>(p[5]),
                reinterpret_cast<decltype(Entry::last_error)>(p[6])};
}

void check(int rc) { TORCH_CHECK(rc == CLIP_OK, "libclip_amd error ", rc, ": ", entry.last_error()); }

int operand_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? CLIP_PRECISION_BF16 : CLIP_PRECISION_F16; }

// [n, H] with unit stride along a row (any row stride)
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 && (r.size(0) < 2 || r.stride(0) >= r.size(1)) ? r : r.contiguous();
}
// [V, H] as the kernels read it: 16-byte aligned rows (a parameter is; anything else is copied.  contiguous() would hand back
// what is contiguous already, wherever it starts and whatever the stride of a single row)
Tensor decoder_of(const Tensor& w) {
  const bool ok = w.stride(1) == 1 && w.stride(0) % 8 == 0 && w.stride(0) >= w.size(1) && w.stride(0) <= (1 << 22) &&
                  reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
  return ok ? w : at::empty(w.sizes(), w.options()).copy_(w);
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
template <typename T = float>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// rows, decoder and targets of one call; labels, or a teacher's values and index
struct Call {
  Tensor rows, weight, bias, labels, values, index;
  int64_t ignore_index;
  double temperature;
  int64_t reduction;
  clip_linear d;
  int32_t k;

  void describe() {
    rows = rows_of(rows);
    weight = decoder_of(weight);
    if (bias.defined()) bias = bias.contiguous();
    k = labels.defined() ? 0 : (int32_t)index.size(1);
    d = clip_linear{operand_of(rows), (int32_t)rows.size(0), (int32_t)rows.size(1), weight.size(0), ptr<uint16_t>(rows), rows.stride(0),
                    ptr<uint16_t>(weight), weight.stride(0), ptr<>(bias)};
  }
  Tensor workspace(int grad) const {
    int64_t bytes = 0;
    check(entry.workspace(&d, k, grad, &bytes));
    return at::empty({bytes}, rows.options().dtype(at::kByte));
  }
  // -> loss, and what the backward pass needs of it: the rows' lse and dev_target
  Tensor forward(Tensor& kept) {
    const c10::DeviceGuard guard(rows.device());
    describe();
    const int64_t n = d.n, kt = k ? 2 * k + 1 : 1;   // floats a row of dev_target
    const auto f32 = rows.options().dtype(at::kFloat);
    // (the loss has storage of its own: a caller may change it in place before the backward pass reads what is kept)
    Tensor loss = reduction == 0 ? at::empty({n}, f32) : at::empty({}, f32);
    kept = at::empty({(reduction == 0 ? 2 + kt : 3 + kt) * n}, f32);
    float *lse = ptr<>(kept), *target = lse + 2 * n, *row_loss = reduction == 0 ? ptr<>(loss) : target + kt * n;
    const Tensor work = workspace(0);
    check(k ? entry.distill(&d, ptr<>(values), ptr<int64_t>(index), k, (float)temperature, (int32_t)reduction, row_loss, lse, target,
                            ptr<>(loss), ptr<void>(work), work.numel(), stream_of(rows))
            : entry.ce(&d, ptr<int64_t>(labels), ignore_index, (int32_t)reduction, row_loss, lse, target, ptr<>(loss), ptr<void>(work),
                       work.numel(), stream_of(rows)));
    return loss;
  }
  void backward(const Tensor& kept, Tensor grad, bool need_h, bool need_w, bool need_b, Tensor& dh, Tensor& dw, Tensor& db) {
    const c10::DeviceGuard guard(rows.device());
    describe();
    const int64_t n = d.n;
    grad = grad.to(at::kFloat).contiguous();
    if (need_h) dh = at::empty(rows.sizes(), rows.options());
    if (need_w) dw = at::empty(weight.sizes(), weight.options());
    if (need_b) db = at::empty({weight.size(0)}, rows.options().dtype(at::kFloat));
    const Tensor work = workspace(1);
    const float *lse = ptr<>(kept), *target = lse + 2 * n;
    const int64_t ld = d.hidden_size;
    check(k ? entry.distill_grad(&d, ptr<int64_t>(index), k, (float)temperature, (int32_t)reduction, lse, target, ptr<>(grad),
                                 ptr<uint16_t>(dh), ld, ptr<uint16_t>(dw), ld, ptr<>(db), ptr<void>(work), work.numel(), stream_of(rows))
            : entry.ce_grad(&d, ptr<int64_t>(labels), ignore_index, (int32_t)reduction, lse, target, ptr<>(grad), ptr<uint16_t>(dh), ld,
                            ptr<uint16_t>(dw), ld, ptr<>(db), ptr<void>(work), work.numel(), stream_of(rows)));
  }
};

struct LinearLoss : torch::autograd::Function<LinearLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& labels,
                        const MaybeTensor& values, const MaybeTensor& index, int64_t ignore_index, double temperature, int64_t reduction) {
    const auto given = [](const MaybeTensor& t) { return t ? *t : Tensor(); };
    Call call{hidden, weight, given(bias), given(labels), given(values), given(index), ignore_index, temperature, reduction, {}, 0};
    Tensor kept;
    Tensor loss = call.forward(kept);
    ctx->save_for_backward({hidden, weight, given(bias), given(labels), given(index), kept});
    ctx->saved_data["args"] = std::vector<double>{(double)reduction, temperature};
    ctx->saved_data["ignore"] = ignore_index;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toDoubleVector();
    const Tensor hidden = saved[0];
    variable_list out(9);
    {
      const at::AutoGradMode off(false);
      Call call{hidden, saved[1], saved[2], saved[3], Tensor(), saved[4], ctx->saved_data["ignore"].toInt(), args[1], (int64_t)args[0], {}, 0};
      Tensor dh;
      call.backward(saved[5], grads[0], ctx->needs_input_grad(0), ctx->needs_input_grad(1), saved[2].defined() && ctx->needs_input_grad(2),
                    dh, out[1], out[2]);
      if (dh.defined()) out[0] = dh.view(hidden.sizes());
    }
    if (at::GradMode::is_enabled()) {   // create_graph: the gradients can be used, but not be differentiated again
      variable_list given;
      for (int i = 0; i < 3; ++i)
        if (out[i].defined()) given.push_back(out[i].detach().requires_grad_());
      const auto error = std::make_shared<torch::autograd::DelayedError>(
          "clip_amd.losses: the gradients cannot be differentiated again", (int64_t)given.size());
      variable_list marked = (*error)(std::move(given));
      for (int i = 0, j = 0; i < 3; ++i)
        if (out[i].defined()) out[i] = marked[j++];
    }
    return out;
  }
};

std::string shape_of(c10::IntArrayRef s) {
  std::ostringstream o;
  o << s;
  return o.str();
}

int64_t reduction_code(const std::string& r) {
  if (r == "mean") return 1;
  if (r == "none") return 0;
  TORCH_CHECK_VALUE(r == "sum", "reduction must be 'none', 'mean' or 'sum', not '", r, "'");
  return 2;
}

// A trace (torch.jit.trace, make_fx) would hold the allocation of the outputs and none of the kernels that fill them
void check_tracing() {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::tracer::impl::is_dispatch_enabled() &&
                                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                              "clip_amd.losses: the calls cannot be traced (torch.compile runs them outside its graphs)");
}

void check_linear(const Tensor& hidden, const Tensor& weight, const MaybeTensor& bias) {
  check_tracing();
  // (the kernels read values only: the tangent of a dual number would be dropped, as if it were zero)
  TORCH_CHECK_NOT_IMPLEMENTED(!isFwGradDefined(hidden) && !isFwGradDefined(weight) && !(bias && isFwGradDefined(*bias)),
                              "clip_amd.losses: no forward-mode derivatives");
  TORCH_CHECK(hidden.is_cuda(), "hidden must be on an MI355X (cuda); clip_amd has no CPU execution path");
  TORCH_CHECK_TYPE((hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf) && weight.scalar_type() == hidden.scalar_type(),
                   "hidden and weight must both be bfloat16 or float16, not ", hidden.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK_VALUE(weight.dim() == 2 && hidden.dim() >= 1 && hidden.size(-1) == weight.size(1), "hidden ", shape_of(hidden.sizes()),
                    " does not fit a [vocab, hidden] weight of ", shape_of(weight.sizes()));
  TORCH_CHECK_VALUE(weight.size(0) >= 1 && weight.size(1) >= 64 && weight.size(1) <= 8192 && weight.size(1) % 64 == 0,
                    "hidden size ", weight.size(1), " (a multiple of 64 up to 8192)");
  const int64_t n = hidden.numel() / weight.size(1);
  TORCH_CHECK_VALUE(n < (1 << 21) && (n + 256) * weight.size(1) < (1ll << 31), n, " rows of ", weight.size(1),
                    " (fewer than 2^21, and 2^31 elements)");
  TORCH_CHECK(weight.device() == hidden.device(), "tensors on ", hidden.device(), " and ", weight.device());
  if (bias) {
    TORCH_CHECK_TYPE(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == weight.size(0), "bias must be float32 [",
                     weight.size(0), "], not ", bias->scalar_type(), " ", shape_of(bias->sizes()));
    TORCH_CHECK(bias->device() == hidden.device(), "tensors on ", hidden.device(), " and ", bias->device());
  }
}

// While a stream is being captured, a leaf whose gradient accumulation node still belongs to a graph of another stream would
// make the backward pass record a wait across streams into the capture, and end the process: refused here, with the reason.
void check_capture(const Tensor& t) {
  if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto stream = node->stream();
  TORCH_CHECK(!stream || *stream == c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device()),
              "clip_amd.losses: a HIP graph is being captured while an earlier loss of the same leaf is still alive (its gradient belongs "
              "to another stream): let go of eager losses before the capture");
}

Tensor apply(const Tensor& hidden, const Tensor& weight, const MaybeTensor& bias, const MaybeTensor& labels, const MaybeTensor& values,
             const MaybeTensor& index, int64_t ignore_index, double temperature, int64_t reduction) {
  const Tensor b = bias ? *bias : Tensor();
  Tensor loss;
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad() || (b.defined() && b.requires_grad()))) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      for (const Tensor* t : {&hidden, &weight, &b}) check_capture(*t);
    loss = LinearLoss::apply(hidden, weight, bias, labels, values, index, ignore_index, temperature, reduction);
  } else {
    const auto given = [](const MaybeTensor& t) { return t ? *t : Tensor(); };
    Call call{hidden, weight, b, given(labels), given(values), given(index), ignore_index, temperature, reduction, {}, 0};
    Tensor kept;
    loss = call.forward(kept);
  }
  return reduction == 0 ? loss.view(hidden.sizes().slice(0, hidden.dim() - 1)) : loss;
}

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const MaybeTensor& bias, const Tensor& labels,
                            int64_t ignore_index, const std::string& reduction) {
  const int64_t code = reduction_code(reduction);
  check_linear(hidden, weight, bias);
  const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
  TORCH_CHECK_VALUE((labels.scalar_type() == at::kLong || labels.scalar_type() == at::kInt) && labels.sizes() == lead,
                    "labels must be integers of shape ", shape_of(lead), ", not ", labels.scalar_type(), " ", shape_of(labels.sizes()));
  TORCH_CHECK(labels.device() == hidden.device(), "tensors on ", hidden.device(), " and ", labels.device());
  const Tensor flat = (labels.dim() == 1 ? labels : labels.reshape({-1})).to(at::kLong).contiguous();
  return apply(hidden, weight, bias, flat, std::nullopt, std::nullopt, ignore_index, 1.0, code);
}

Tensor linear_distillation(const Tensor& hidden, const Tensor& weight, const MaybeTensor& bias, const Tensor& values, const Tensor& index,
                           double temperature, const std::string& reduction) {
  const int64_t code = reduction_code(reduction);
  check_linear(hidden, weight, bias);
  const auto lead = hidden.sizes().slice(0, hidden.dim() - 1);
  TORCH_CHECK_VALUE(index.scalar_type() == at::kLong && index.dim() == hidden.dim() && index.sizes().slice(0, index.dim() - 1) == lead &&
                        values.sizes() == index.sizes() && values.is_floating_point(),
                    "teacher values / index must be floating point / int64 of shape ", shape_of(lead), " + [k], not ", values.scalar_type(), " ",
                    shape_of(values.sizes()), " / ", index.scalar_type(), " ", shape_of(index.sizes()));
  const int64_t k = index.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= 1024, k, " teacher entries per row (1 .. 1024)");
  // (its square and its reciprocal stay numbers in fp32)
  TORCH_CHECK_VALUE(temperature >= 1e-6 && temperature <= 1e6, "temperature must be between 1e-6 and 1e6, not ", temperature);
  for (const Tensor* t : {&values, &index}) TORCH_CHECK(t->device() == hidden.device(), "tensors on ", hidden.device(), " and ", t->device());
  return apply(hidden, weight, bias, std::nullopt, values.detach().to(at::kFloat).reshape({-1, k}).contiguous(), index.reshape({-1, k}).contiguous(), 0,
               temperature, code);
}

std::tuple<Tensor, Tensor> topk_logits(const Tensor& logits, int64_t k) {
  check_tracing();
  TORCH_CHECK(logits.is_cuda(), "logits must be on an MI355X (cuda); clip_amd has no CPU execution path");
  const auto type = logits.scalar_type();
  TORCH_CHECK_TYPE((type == at::kFloat || type == at::kBFloat16 || type == at::kHalf) && logits.dim() >= 1,
                   "logits must be float32, bfloat16 or float16 with at least one dimension, not ", type);
  const int64_t vocab = logits.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= std::min<int64_t>(vocab, 1024) && vocab <= INT32_MAX, "k = ", k, " of ", vocab,
                    " scores (1 .. min(vocab, 1024))");
  const Tensor rows = rows_of(logits.detach());
  TORCH_CHECK_VALUE(rows.size(0) <= INT32_MAX, "more than 2^31 - 1 rows");
  const c10::DeviceGuard guard(logits.device());
  auto shape = logits.sizes().vec();
  shape.back() = k;
  Tensor values = at::empty(shape, rows.options()), index = at::empty(shape, rows.options().dtype(at::kLong));
  check(entry.topk(type == at::kFloat ? CLIP_PRECISION_FP32 : operand_of(rows), ptr<void>(rows), rows.stride(0), (int32_t)rows.size(0),
                   (int32_t)vocab, (int32_t)k, ptr<void>(values), ptr<int64_t>(index), stream_of(rows)));
  return {values, index};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", torch::wrap_pybind_function(bind));
  m.def("linear_cross_entropy", torch::wrap_pybind_function_no_gil(linear_cross_entropy));
  m.def("linear_distillation", torch::wrap_pybind_function_no_gil(linear_distillation));
  m.def("topk_logits", torch::wrap_pybind_function_no_gil(topk_logits));
}
