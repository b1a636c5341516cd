// PyTorch side of the query adapter: differentiable layer norm, linear layer and
// preference loss over the C ABI (include/cvs.h). Shapes are checked here (shape and
// value faults raise ValueError, dtypes TypeError, everything else RuntimeError);
// workspaces, kept statistics and results come from torch's allocator on the current
// stream of the inputs' device. First derivatives only.
#include "torch_adapter.h"

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

#include <cstdint>
#include <optional>

#include "cvs.h"

namespace cvs_torch {
namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void check(cvs_status s, const char* what) { TORCH_CHECK(s == CVS_OK, what, ": ", cvs_last_error()); }

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
const void* ptr(const OptTensor& t) { return given(t) ? t->data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

int code(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat: return CVS_F32;
    case torch::kHalf: return CVS_F16;
    case torch::kBFloat16: return CVS_BF16;
    default: return -1;
  }
}

int64_t pad8(int64_t v) { return (v + 7) / 8 * 8; }
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : pad8(t.size(1)); }

// An uninitialised tensor on the device of `like`, without a trip through the
// dispatcher (a training pass makes up to eight; each trip costs most of a microsecond).
Tensor fresh(at::IntArrayRef sizes, torch::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

Tensor bytes(size_t n, const Tensor& like) {
  return fresh({static_cast<int64_t>(std::max<size_t>(n, 256))}, torch::kUInt8, like);
}

// A 2-D tensor whose rows are contiguous; rows may be any distance apart.
Tensor with_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1 ? t : t.contiguous(); }

// Rows the tensor-memory accelerator can read as they are.
bool tiles_ok(const Tensor& t) {
  return reinterpret_cast<std::uintptr_t>(t.data_ptr()) % 16 == 0 && (t.stride(1) == 1 || t.size(1) <= 1) &&
         (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)));
}

// The same with rows the tensor-memory accelerator can read: 16-byte aligned,
// otherwise copied into rows padded to a multiple of 8 elements.
Tensor with_tiles(const Tensor& t) {
  if (tiles_ok(t)) return t;
  const Tensor src = with_rows(t);
  const Tensor out = fresh({t.size(0), pad8(t.size(1))}, t.scalar_type(), t);
  check(cvs_align_rows(src.data_ptr(), row_stride(src), code(src), src.size(0), static_cast<int>(src.size(1)), out.data_ptr(),
                       out.size(1), stream_of(src)),
        "linear");
  return out.narrow(1, 0, t.size(1));
}

void check_device(const Tensor& t, const char* name, const Tensor& first) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == first.device(), name, " must be on the same device as the input");
}

// A leaf whose gradient accumulator was made on the default stream (by a graph that is
// still alive) would make a captured backward pass wait for that stream, which cannot take
// part in a capture: that ends it and, from the autograd thread, the process. Refused
// before that. (Another stream's accumulator, a warm-up's, joins the capture.)
void check_capture(std::initializer_list<const Tensor*> inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream.has_value() || *stream != c10::cuda::getDefaultCUDAStream(t->device().index()).unwrap(),
                "a parameter of a captured backward pass still belongs to an autograd graph made on another stream, "
                "the default one; release that graph's outputs before the capture, or run it on another stream");
  }
}

// The operators have no forward-mode derivative: an input's tangent would be lost.
void check_tangents(std::initializer_list<const Tensor*> inputs, const char* what) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what,
                ": forward-mode derivatives (torch.autograd.forward_ad) are not supported");
}

bool wants_grad(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

void first_order_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "the adapter's operators have no second derivative (create_graph=True)");
}

// What a backward pass has to know besides its tensors, in one number: a small code
// (the weights' type, the activation) and which inputs there were.
constexpr int64_t kHasWeight = 1 << 8, kHasBias = 1 << 9, kHasResidual = 1 << 10;

Tensor or_undefined(const OptTensor& t) { return given(t) ? *t : Tensor(); }

// Number of rows of a tensor seen as [rows, width].
Tensor flat(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)}); }

// ---- layer norm -------------------------------------------------------------
struct NormOut {
  Tensor y, mean, rstd;
};

NormOut norm_forward(const Tensor& x_in, const Tensor& weight, const Tensor& bias, double eps, bool keep) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = with_rows(x_in);
  const int64_t rows = x.size(0), d = x.size(1);
  NormOut out;
  out.y = fresh({rows, d}, x.scalar_type(), x);
  if (keep) {
    out.mean = fresh({rows}, torch::kFloat, x);
    out.rstd = fresh({rows}, torch::kFloat, x);
  }
  const Tensor& any = weight.defined() ? weight : bias;
  const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  check(cvs_layer_norm(x.data_ptr(), code(x), rows, static_cast<int>(d), row_stride(x),
                       w.defined() ? w.data_ptr() : nullptr, b.defined() ? b.data_ptr() : nullptr,
                       any.defined() ? code(any) : code(x), static_cast<float>(eps), out.y.data_ptr(), d,
                       keep ? out.mean.data_ptr<float>() : nullptr, keep ? out.rstd.data_ptr<float>() : nullptr,
                       stream_of(x)),
        "layer_norm");
  return out;
}

class LayerNormFn : public torch::autograd::Function<LayerNormFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    NormOut out = norm_forward(x, or_undefined(weight), or_undefined(bias), eps, true);
    ctx->save_for_backward({x, or_undefined(weight), out.mean, out.rstd});
    const int64_t type = given(bias) ? code(*bias) : (given(weight) ? code(*weight) : code(x));
    ctx->saved_data["layer"] = type | (given(weight) ? kHasWeight : 0) | (given(bias) ? kHasBias : 0);
    return out.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor x = with_rows(saved[0]), dy = with_rows(grads[0]);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t layer = ctx->saved_data["layer"].toInt();
    const bool has_w = layer & kHasWeight, has_b = layer & kHasBias;
    const int type = static_cast<int>(layer & 0xff);
    const Tensor w = has_w ? saved[1].contiguous() : Tensor();
    const int64_t rows = x.size(0), d = x.size(1);
    const auto wtype = type == CVS_F32 ? torch::kFloat : x.scalar_type();
    size_t edge = 1;
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = fresh({rows, d}, x.scalar_type(), x);
    if (has_w && ctx->needs_input_grad(edge++)) dw = fresh({d}, wtype, x);
    if (has_b && ctx->needs_input_grad(edge++)) db = fresh({d}, wtype, x);
    size_t need = 0;
    Tensor ws;
    if (dw.defined() || db.defined()) {
      check(cvs_layer_norm_backward_workspace_size(rows, static_cast<int>(d), &need), "layer_norm");
      ws = bytes(need, x);
    }
    check(cvs_layer_norm_backward(dy.data_ptr(), row_stride(dy), x.data_ptr(), code(x), rows, static_cast<int>(d),
                                  row_stride(x), has_w ? w.data_ptr() : nullptr, type, saved[2].data_ptr<float>(),
                                  saved[3].data_ptr<float>(), dx.defined() ? dx.data_ptr() : nullptr, d,
                                  dw.defined() ? dw.data_ptr() : nullptr, db.defined() ? db.data_ptr() : nullptr,
                                  ws.defined() ? ws.data_ptr() : nullptr, need, stream_of(x)),
          "layer_norm");
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK(x.is_cuda(), "layer_norm: x must be a CUDA tensor");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= CVS_MAX_NORM_WIDTH,
                    "layer_norm: the last dimension must be in 1 .. ", CVS_MAX_NORM_WIDTH);
  TORCH_CHECK_TYPE(code(x) >= 0, "layer_norm: x must be float32, float16 or bfloat16, not ", x.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative");
  for (const OptTensor* t : {&weight, &bias}) {
    if (!given(*t)) continue;
    check_device(**t, "layer_norm: weight and bias", x);
    TORCH_CHECK_VALUE((*t)->dim() == 1 && (*t)->size(0) == x.size(-1), "layer_norm: weight and bias must be [", x.size(-1), "]");
    TORCH_CHECK_TYPE((*t)->scalar_type() == x.scalar_type() || (*t)->scalar_type() == torch::kFloat,
                     "layer_norm: weight and bias must be float32 or of x's dtype");
  }
  if (given(weight) && given(bias))
    TORCH_CHECK_TYPE(weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias must have one dtype");
  const Tensor w = or_undefined(weight), b = or_undefined(bias);
  check_tangents({&x, &w, &b}, "layer_norm");
  Tensor y;
  if (wants_grad({&x, &w, &b})) {
    check_capture({&x, &w, &b});
    y = LayerNormFn::apply(flat(x), weight, bias, eps);
  } else {
    y = norm_forward(flat(x), w, b, eps, false).y;
  }
  return x.dim() == 2 ? y : y.reshape(x.sizes());
}

// ---- linear -----------------------------------------------------------------
struct LinearOut {
  Tensor y, z;
  Tensor x, w;  // as the product read them (copies where their rows were not aligned)
};

LinearOut linear_forward(const Tensor& x_in, const Tensor& w_in, const Tensor& bias_in, const Tensor& residual_in,
                         int activation, bool keep) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const int64_t m = x_in.size(0), k = x_in.size(1), n = w_in.size(0);
  const bool small = m <= CVS_LINEAR_SMALL_ROWS;
  const Tensor x = small ? with_rows(x_in) : with_tiles(x_in);
  Tensor w = small ? with_rows(w_in) : with_tiles(w_in);
  if (small && w.size(0) > 1 && w.stride(0) < k) w = w.contiguous();
  const Tensor bias = bias_in.defined() ? bias_in.contiguous() : bias_in;
  const Tensor residual = residual_in.defined() ? with_rows(residual_in) : residual_in;
  LinearOut out;
  out.y = fresh({m, n}, x.scalar_type(), x);
  if (keep) out.z = fresh({m, pad8(n)}, torch::kHalf, x);
  check(cvs_linear(x.data_ptr(), row_stride(x), w.data_ptr(), row_stride(w), bias.defined() ? bias.data_ptr() : nullptr,
                   residual.defined() ? residual.data_ptr() : nullptr, residual.defined() ? row_stride(residual) : 0,
                   activation, code(x), m, static_cast<int>(n), static_cast<int>(k), out.y.data_ptr(), n,
                   keep ? out.z.data_ptr() : nullptr, keep ? pad8(n) : 0, stream_of(x)),
        "linear");
  out.x = x;
  out.w = w;
  return out;
}

class LinearFn : public torch::autograd::Function<LinearFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                        const OptTensor& residual, int64_t activation) {
    // z is only read by an activation's derivative.
    const bool keep = activation != CVS_ACT_NONE;
    LinearOut out = linear_forward(x, weight, or_undefined(bias), or_undefined(residual), static_cast<int>(activation), keep);
    // Where the product read aligned copies, the backward pass reads them again instead
    // of making its own (more than CVS_LINEAR_SMALL_ROWS rows; else the inputs as they are).
    ctx->save_for_backward({out.x, out.w, out.z});
    ctx->saved_data["layer"] = activation | (given(bias) ? kHasBias : 0) | (given(residual) ? kHasResidual : 0);
    return out.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const int64_t layer = ctx->saved_data["layer"].toInt();
    const bool has_b = layer & kHasBias, has_r = layer & kHasResidual;
    const int activation = static_cast<int>(layer & 0xff);
    const c10::cuda::CUDAGuard guard(saved[0].device());
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    size_t edge = 2;
    const bool need_b = has_b && ctx->needs_input_grad(edge++);
    const bool need_r = has_r && ctx->needs_input_grad(edge++);
    const Tensor& z = saved[2];
    const int64_t m = saved[0].size(0), k = saved[0].size(1), n = saved[1].size(0);
    Tensor dx, dw, db;
    if (need_x) dx = fresh({m, k}, saved[0].scalar_type(), saved[0]);
    if (need_w) dw = fresh({n, k}, saved[0].scalar_type(), saved[0]);
    if (need_b) db = fresh({n}, saved[0].scalar_type(), saved[0]);
    if (need_x || need_w || need_b) {
      const Tensor dy = with_rows(grads[0]);
      const Tensor x = need_w ? with_tiles(saved[0]) : saved[0], w = need_x ? with_tiles(saved[1]) : saved[1];
      size_t need = 0;
      check(cvs_linear_backward_workspace_size(activation, m, static_cast<int>(n), static_cast<int>(k), &need), "linear");
      if (activation == CVS_ACT_NONE && tiles_ok(dy)) need -= (static_cast<size_t>(m) * pad8(n) * 2 + 255) / 256 * 256;
      const Tensor ws = bytes(need, dy);
      check(cvs_linear_backward(dy.data_ptr(), row_stride(dy), x.data_ptr(), row_stride(x), w.data_ptr(), row_stride(w),
                                z.defined() ? z.data_ptr() : nullptr, z.defined() ? z.size(1) : 0, activation, code(dy),
                                m, static_cast<int>(n), static_cast<int>(k), need_x ? dx.data_ptr() : nullptr, k,
                                need_w ? dw.data_ptr() : nullptr, k, need_b ? db.data_ptr() : nullptr, ws.data_ptr(),
                                need, stream_of(dy)),
            "linear");
    }
    return {dx, dw, db, need_r ? grads[0] : Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t activation,
              const OptTensor& residual) {
  TORCH_CHECK(x.is_cuda(), "linear: x must be a CUDA tensor");
  TORCH_CHECK_TYPE(x.scalar_type() == torch::kHalf || x.scalar_type() == torch::kBFloat16,
                   "linear: x must be float16 or bfloat16, not ", x.scalar_type());
  check_device(weight, "linear: weight", x);
  TORCH_CHECK_TYPE(weight.scalar_type() == x.scalar_type(), "linear: weight must have x's dtype");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1 &&
                        weight.size(0) <= CVS_MAX_LAYER_WIDTH && weight.size(1) <= CVS_MAX_LAYER_WIDTH,
                    "linear: weight must be [n, k], both at most ", CVS_MAX_LAYER_WIDTH);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == weight.size(1), "linear: x must be [..., ", weight.size(1), "]");
  TORCH_CHECK_VALUE(activation >= CVS_ACT_NONE && activation <= CVS_ACT_SILU, "linear: unknown activation");
  const int64_t n = weight.size(0);
  if (given(bias)) {
    check_device(*bias, "linear: bias", x);
    TORCH_CHECK_TYPE(bias->scalar_type() == x.scalar_type(), "linear: bias must have x's dtype");
    TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "linear: bias must be [", n, "]");
  }
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  if (given(residual)) {
    check_device(*residual, "linear: residual", x);
    TORCH_CHECK_TYPE(residual->scalar_type() == x.scalar_type(), "linear: residual must have x's dtype");
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(shape), "linear: residual must have the result's shape ",
                      at::IntArrayRef(shape));
  }
  const Tensor b = or_undefined(bias), r = or_undefined(residual);
  check_tangents({&x, &weight, &b, &r}, "linear");
  const Tensor r2 = r.defined() ? flat(r) : r;
  Tensor y;
  if (wants_grad({&x, &weight, &b, &r})) {
    check_capture({&x, &weight, &b, &r});
    y = LinearFn::apply(flat(x), weight, bias, r.defined() ? OptTensor(r2) : OptTensor(), activation);
  } else {
    y = linear_forward(flat(x), weight, b, r2, static_cast<int>(activation), false).y;
  }
  return x.dim() == 2 ? y : y.reshape(shape);
}

// ---- preference loss ----------------------------------------------------------
struct PreferenceOut {
  Tensor loss, weight, margins, grad;
};

PreferenceOut preference_forward(const Tensor& q_in, const Tensor& ref_in, const Tensor& chosen_in,
                                 const Tensor& rejected_in, const Tensor& corpus, bool cosine, double scale,
                                 double smoothing, bool mean, bool keep) {
  const c10::cuda::CUDAGuard guard(corpus.device());
  const Tensor q = with_rows(q_in), ref = ref_in.defined() ? with_rows(ref_in) : ref_in;
  const Tensor chosen = chosen_in.contiguous(), rejected = with_rows(rejected_in);
  const int64_t b = q.size(0), d = q.size(1), r = rejected.size(1);
  PreferenceOut out;
  out.loss = fresh({}, torch::kFloat, corpus);
  out.weight = fresh({}, torch::kFloat, corpus);
  out.margins = fresh({b, r}, torch::kFloat, corpus);
  if (keep) out.grad = fresh({b, pad8(d)}, torch::kFloat, corpus);
  size_t need = 0;
  check(cvs_preference_loss_workspace_size(b, static_cast<int>(r), &need), "preference_loss");
  const Tensor ws = bytes(need, corpus);
  check(cvs_preference_loss(q.data_ptr(), code(q), row_stride(q), ref.defined() ? ref.data_ptr() : nullptr,
                            ref.defined() ? code(ref) : CVS_F32, ref.defined() ? row_stride(ref) : 0, b,
                            static_cast<int>(d), cosine ? 1 : 0, corpus.data_ptr(), corpus.size(0),
                            static_cast<int>(corpus.size(1)), chosen.data_ptr<int64_t>(), rejected.data_ptr<int64_t>(),
                            row_stride(rejected), static_cast<int>(r), static_cast<float>(scale),
                            static_cast<float>(smoothing), mean ? 1 : 0, out.loss.data_ptr<float>(),
                            out.weight.data_ptr<float>(), out.margins.data_ptr<float>(),
                            keep ? out.grad.data_ptr<float>() : nullptr, pad8(d), ws.data_ptr(), need, stream_of(corpus)),
        "preference_loss");
  return out;
}

class PreferenceFn : public torch::autograd::Function<PreferenceFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& ref, const Tensor& chosen,
                               const Tensor& rejected, const Tensor& corpus, bool cosine, double scale,
                               double smoothing, bool mean) {
    PreferenceOut out = preference_forward(q, or_undefined(ref), chosen, rejected, corpus, cosine, scale, smoothing, mean, true);
    ctx->save_for_backward({out.grad, out.weight});
    ctx->saved_data["width"] = q.size(1);
    ctx->saved_data["type"] = static_cast<int64_t>(q.scalar_type());
    ctx->mark_non_differentiable({out.margins});
    return {out.loss, out.margins};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor& grad = saved[0];
    const c10::cuda::CUDAGuard guard(grad.device());
    const int64_t b = grad.size(0), d = ctx->saved_data["width"].toInt();
    const auto type = static_cast<torch::ScalarType>(ctx->saved_data["type"].toInt());
    const Tensor upstream = grads[0].to(torch::kFloat);
    Tensor dq = fresh({b, d}, type, grad);
    check(cvs_preference_grad(grad.data_ptr<float>(), grad.size(1), b, static_cast<int>(d), saved[1].data_ptr<float>(),
                              upstream.data_ptr<float>(), code(dq), dq.data_ptr(), stream_of(grad)),
          "preference_loss");
    return {dq, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> preference_loss(const Tensor& q, const OptTensor& reference, const Tensor& chosen,
                                           const Tensor& rejected, const Tensor& corpus, bool cosine, double scale,
                                           double smoothing, bool mean) {
  TORCH_CHECK(corpus.is_cuda(), "preference_loss: the corpus must be a CUDA tensor");
  TORCH_CHECK(corpus.dim() == 2 && corpus.is_contiguous() && corpus.scalar_type() == torch::kHalf,
              "preference_loss: the corpus must be a contiguous float16 matrix");
  check_device(q, "preference_loss: queries", corpus);
  TORCH_CHECK_VALUE(q.dim() == 2 && q.size(1) >= 1 && q.size(1) <= corpus.size(1),
                    "preference_loss: queries must be [b, d], no wider than the corpus");
  TORCH_CHECK_TYPE(code(q) >= 0, "preference_loss: queries must be float32, float16 or bfloat16, not ", q.scalar_type());
  const Tensor ref = given(reference) ? reference->detach() : Tensor();
  if (ref.defined()) {
    check_device(ref, "preference_loss: reference", corpus);
    TORCH_CHECK_VALUE(ref.sizes() == q.sizes(), "preference_loss: reference must have the queries' shape");
    TORCH_CHECK_TYPE(code(ref) >= 0, "preference_loss: reference must be float32, float16 or bfloat16");
  }
  check_device(chosen, "preference_loss: chosen", corpus);
  check_device(rejected, "preference_loss: rejected", corpus);
  TORCH_CHECK_TYPE(chosen.scalar_type() == torch::kLong && rejected.scalar_type() == torch::kLong,
                   "preference_loss: chosen and rejected must be int64 row ids");
  TORCH_CHECK_VALUE(chosen.dim() == 1 && chosen.size(0) == q.size(0), "preference_loss: chosen must be [b]");
  TORCH_CHECK_VALUE(rejected.dim() == 2 && rejected.size(0) == q.size(0) && rejected.size(1) >= 1 &&
                        rejected.size(1) <= CVS_MAX_REJECTED,
                    "preference_loss: rejected must be [b] or [b, r] with r in 1 .. ", CVS_MAX_REJECTED);
  TORCH_CHECK_VALUE(smoothing >= 0 && smoothing <= 1, "preference_loss: label_smoothing must be in 0 .. 1");
  check_tangents({&q}, "preference_loss");
  if (wants_grad({&q})) {
    check_capture({&q});
    const auto out = PreferenceFn::apply(q, ref.defined() ? OptTensor(ref) : OptTensor(), chosen, rejected, corpus, cosine,
                                         scale, smoothing, mean);
    return {out[0], out[1]};
  }
  const PreferenceOut out = preference_forward(q, ref, chosen, rejected, corpus, cosine, scale, smoothing, mean, false);
  return {out.loss, out.margins};
}

}  // namespace

void bind_adapter(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm, "Layer norm over the last dimension (differentiable)", py::arg("x"),
        py::arg("weight"), py::arg("bias"), py::arg("eps"));
  m.def("linear", &linear, "act(x w^T + bias) + residual (differentiable)", py::arg("x"), py::arg("weight"),
        py::arg("bias"), py::arg("activation"), py::arg("residual"));
  m.def("preference_loss", &preference_loss, "Preference loss over corpus rows (differentiable): loss, margins",
        py::arg("q"), py::arg("reference"), py::arg("chosen"), py::arg("rejected"), py::arg("corpus"),
        py::arg("cosine"), py::arg("scale"), py::arg("label_smoothing"), py::arg("mean"));
}

}  // namespace cvs_torch
