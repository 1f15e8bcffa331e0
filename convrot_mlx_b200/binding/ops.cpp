// Torch-side entry points of the 8-bit and training operators: argument
// checks, output allocation, autograd nodes and the call of the C ABI
// (include/convrot_b200.h), in C++ so that a small call is not bound by the
// interpreter and a backward pass needs no interpreter at all.  The Python
// modules int8, rotary, norm and activation hold the public functions and
// their documentation; everything they refuse is refused here.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <vector>

#include "convrot_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kPitch = 16;        // rows of codes start on multiples of 16 bytes
constexpr int64_t kMaxDot = 131072;   // products that one int32 dot can sum
constexpr int64_t kSavedGroup = 128;  // features of a row that share one scale of a saved GELU input

// --- errors -------------------------------------------------------------

template <typename... Args>
[[noreturn]] void refuse(Args&&... args) {
  throw py::value_error(c10::str(std::forward<Args>(args)...));
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

// The exception that _lib.check raises for a status; plain in a thread of the
// autograd engine, which holds no interpreter.
void check(int status, const char* what) {
  if (status == CONVROT_OK) return;
  const std::string message = convrot_last_error();
  if (!PyGILState_Check()) throw std::runtime_error(c10::str(what, ": ", message));
  if (status == CONVROT_ERR_INVALID) throw py::value_error(message);
  const std::string whole = c10::str(what, ": ", message);
  if (status == CONVROT_ERR_UNSUPPORTED) {
    PyErr_SetString(PyExc_NotImplementedError, whole.c_str());
  } else {
    const py::object type = py::module_::import("convrot_mlx_b200._lib").attr("ConvRotError");
    PyErr_SetString(type.ptr(), whole.c_str());
  }
  throw py::error_already_set();
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return CONVROT_BF16;
    case at::kHalf: return CONVROT_F16;
    case at::kFloat: return CONVROT_F32;
    default: refuse("unsupported dtype ", t, "; expected float32, float16 or bfloat16");
  }
}

// All tensors of a call (undefined ones aside) on the device of the first.
void require_cuda(std::initializer_list<const Tensor*> tensors) {
  const c10::Device home = (*tensors.begin())->device();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (!t->is_cuda())
      refuse("convrot_mlx_b200 runs on CUDA (sm_100a) only; got a tensor on ", t->device().str(),
             " (there is no CPU fallback)");
    if (t->device() != home) refuse("expected all tensors on ", home.str(), ", got one on ", t->device().str());
  }
}

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "the gradient of ", what,
              " cannot itself be differentiated (create_graph is not supported)");
}

// Forward-mode derivatives are not formed: a tangent would be dropped, and the
// output read as constant.
void no_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors) {
    if (!t->defined() || !t->_fw_grad(/*level=*/0).defined()) continue;
    PyErr_SetString(PyExc_NotImplementedError,
                    c10::str("the forward-mode derivative of ", what, " is not supported").c_str());
    throw py::error_already_set();
  }
}

// --- small helpers --------------------------------------------------------

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
Tensor or_undefined(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

Tensor f32_vector(const Tensor& t) {
  return !t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous()) ? t : t.to(at::kFloat).contiguous();
}

// x as (rows, features) with unit stride along the features and rows that do
// not overlap.
Tensor rows_of(const Tensor& x) {
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if (r.stride(1) != 1 || r.stride(0) < r.size(1)) {
    r = r.contiguous();
    if (r.stride(0) < r.size(1)) r = r.as_strided(r.sizes(), {r.size(1), 1});  // a single row
  }
  return r;
}

Tensor padded_rows(const Tensor& codes) {
  if (codes.stride(1) == 1 && codes.stride(0) >= codes.size(1) && codes.stride(0) % kPitch == 0 &&
      reinterpret_cast<uintptr_t>(codes.data_ptr()) % kPitch == 0)
    return codes;
  const int64_t pitch = (codes.size(1) + kPitch - 1) / kPitch * kPitch;
  Tensor out = at::empty({codes.size(0), pitch}, codes.options()).narrow(1, 0, codes.size(1));
  out.copy_(codes);
  return out;
}

// --- 8-bit linear -----------------------------------------------------------

// The quantizer and the product in one call; n columns out.
Tensor i8_product(const Tensor& x, const Tensor& col_scale, const Tensor& qweight, int layout, const Tensor& wscales,
                  const Tensor& bias, int64_t n) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const Tensor r = rows_of(x);
  const int64_t m = r.size(0), k = r.size(1), pitch = (k + kPitch - 1) / kPitch * kPitch;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  const Tensor out = at::empty(shape, x.options());
  const Tensor space = at::empty({m * (pitch + 4)}, qweight.options());  // codes, then scales
  auto* codes = static_cast<int8_t*>(space.data_ptr());
  const int dtype = dtype_code(x.scalar_type());
  check(convrot_i8_linear(r.data_ptr(), dtype, r.stride(0), static_cast<const float*>(address(col_scale)),
                          static_cast<const int8_t*>(qweight.data_ptr()), qweight.stride(0), layout,
                          static_cast<const float*>(address(wscales)), static_cast<const float*>(address(bias)),
                          out.data_ptr(), dtype, m, n, k, codes, pitch, reinterpret_cast<float*>(codes + m * pitch),
                          stream_of(x)),
        "convrot_i8_linear");
  return out;
}

// The gradient of the input over more channels k than one int32 dot can sum:
// the codes are formed once for the whole token, each range of kMaxDot channels
// is an exact dot, and the ranges' products are added in float32, in order.
Tensor i8_gradient_in_ranges(const Tensor& dy, const Tensor& wscales, const Tensor& qweight) {
  const c10::cuda::OptionalCUDAGuard guard(dy.device());
  const Tensor r = rows_of(dy);
  const int64_t m = r.size(0), k = r.size(1), n = qweight.size(1), pitch = (k + kPitch - 1) / kPitch * kPitch;
  std::vector<int64_t> shape(dy.sizes().begin(), dy.sizes().end());
  shape.back() = n;
  const Tensor codes = at::empty({m, pitch}, qweight.options()), scales = at::empty({m}, wscales.options());
  check(convrot_quantize_i8(r.data_ptr(), dtype_code(r.scalar_type()), m, k, r.stride(0),
                            static_cast<const float*>(wscales.data_ptr()), static_cast<int8_t*>(codes.data_ptr()), pitch,
                            static_cast<float*>(scales.data_ptr()), stream_of(dy)),
        "convrot_quantize_i8");
  Tensor sum;
  for (int64_t at = 0; at < k; at += kMaxDot) {
    const Tensor part = at::empty(shape, scales.options());
    check(convrot_i8_gemm(static_cast<const int8_t*>(codes.data_ptr()) + at, pitch,
                          static_cast<const int8_t*>(qweight.data_ptr()) + at * qweight.stride(0), qweight.stride(0),
                          CONVROT_LAYOUT_KN, static_cast<const float*>(scales.data_ptr()), nullptr, nullptr,
                          part.data_ptr(), CONVROT_F32, m, n, std::min(kMaxDot, k - at), stream_of(dy)),
          "convrot_i8_gemm");
    sum = sum.defined() ? sum.add_(part) : part;
  }
  return sum.to(dy.scalar_type());
}

struct Int8Linear : torch::autograd::Function<Int8Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& qweight, const Tensor& wscales,
                        const std::optional<Tensor>& bias) {
    ctx->save_for_backward({qweight, wscales});
    return i8_product(x, {}, qweight, CONVROT_LAYOUT_NK, wscales, or_undefined(bias), qweight.size(0));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("int8_linear");
    const auto saved = ctx->get_saved_variables();
    const Tensor &qweight = saved[0], &wscales = saved[1];
    if (qweight.size(0) > kMaxDot) return {i8_gradient_in_ranges(grads[0], wscales, qweight), {}, {}, {}};
    return {i8_product(grads[0], wscales, qweight, CONVROT_LAYOUT_KN, {}, {}, qweight.size(1)), {}, {}, {}};
  }
};

Tensor int8_linear(const Tensor& x, const Tensor& qweight, const Tensor& wscales, const std::optional<Tensor>& bias) {
  if (x.dim() == 0) refuse("int8 linear expects at least one dimension");
  if (qweight.dim() != 2 || qweight.scalar_type() != at::kChar)
    refuse("int8 weight must be a 2D int8 tensor, got ", shape_of(qweight), " ", qweight.scalar_type());
  const int64_t n = qweight.size(0), k = x.size(-1);
  if (qweight.size(1) != k || k == 0)
    refuse("int8 weight must be (N, K) rows; activation K=", k, ", weight=", shape_of(qweight));
  if (wscales.dim() != 1 || wscales.size(0) != n)
    refuse("int8 weight scales must have shape (", n, ",), got ", shape_of(wscales));
  const Tensor b = or_undefined(bias);
  if (b.defined() && (b.dim() != 1 || b.size(0) != n))
    refuse("int8 bias must have shape (", n, ",), got ", shape_of(b));
  if (wants_grad(wscales) || wants_grad(b))
    refuse("the weight scales and the bias of an int8 linear are frozen: they may not require gradients");
  dtype_code(x.scalar_type());
  no_tangents("int8_linear", {&x, &wscales, &b});
  require_cuda({&x, &qweight, &wscales, &b});
  const Tensor w = padded_rows(qweight), ws = f32_vector(wscales), fb = f32_vector(b);
  if (at::GradMode::is_enabled() && x.requires_grad())
    return Int8Linear::apply(x, w, ws, fb.defined() ? std::optional<Tensor>(fb) : std::nullopt);
  return i8_product(x, {}, w, CONVROT_LAYOUT_NK, ws, fb, n);
}

// --- rotary -------------------------------------------------------------------

struct RotaryHow {
  std::vector<int32_t> widths;
  double theta;
  bool interleaved;
};

Tensor unit_stride(const Tensor& t) { return !t.defined() || t.stride(3) == 1 ? t : t.contiguous(); }

// q, k (either may be undefined) turned into new tensors, packed as (batch,
// heads, tokens, dim), or with the heads inside the tokens.
std::pair<Tensor, Tensor> turn(const Tensor& q_in, const Tensor& k_in, const Tensor& positions, const RotaryHow& how,
                               bool inverse, bool heads_inside) {
  const Tensor q = unit_stride(q_in), k = unit_stride(k_in);
  const Tensor& any = q.defined() ? q : k;
  const c10::cuda::OptionalCUDAGuard guard(any.device());
  const int64_t b = any.size(0), t = any.size(2), d = any.size(3);
  int64_t strides[12] = {};
  Tensor out[2];
  int64_t heads[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    const Tensor& in = i ? k : q;
    if (!in.defined()) continue;
    const int64_t h = heads[i] = in.size(1);
    out[i] = heads_inside ? at::empty({b, t, h, d}, in.options()).transpose(1, 2) : at::empty({b, h, t, d}, in.options());
    for (int s = 0; s < 3; ++s) {
      strides[6 * i + s] = in.stride(s);
      strides[6 * i + 3 + s] = out[i].stride(s);
    }
  }
  check(convrot_axial_rotary(dtype_code(any.scalar_type()), b, t, d, address(q), address(out[0]), heads[0], address(k),
                             address(out[1]), heads[1], strides, static_cast<const float*>(positions.data_ptr()),
                             positions.dim() == 3 ? positions.stride(0) : 0, static_cast<int>(how.widths.size()),
                             how.widths.data(), how.theta, how.interleaved, inverse, stream_of(any)),
        "convrot_axial_rotary");
  return {out[0], out[1]};
}

struct AxialRotary : torch::autograd::Function<AxialRotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const std::optional<Tensor>& k,
                               const Tensor& positions, const RotaryHow& how) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions});
    ctx->saved_data["widths"] = std::vector<int64_t>(how.widths.begin(), how.widths.end());
    ctx->saved_data["theta"] = how.theta;
    ctx->saved_data["interleaved"] = how.interleaved;
    // the gradients take the memory order of the inputs, often columns of one projection's output
    ctx->saved_data["heads_inside"] = q.stride(1) < q.stride(2);
    const auto [yq, yk] = turn(q, or_undefined(k), positions, how, false, false);
    if (yk.defined()) return {yq, yk};
    return {yq};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("axial_rotary");
    RotaryHow how;
    for (int64_t w : ctx->saved_data["widths"].toIntVector()) how.widths.push_back(static_cast<int32_t>(w));
    how.theta = ctx->saved_data["theta"].toDouble();
    how.interleaved = ctx->saved_data["interleaved"].toBool();
    const Tensor dk = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dk.defined()) return {{}, {}, {}, {}};
    const auto [gq, gk] = turn(grads[0], dk, ctx->get_saved_variables()[0], how, true,
                               ctx->saved_data["heads_inside"].toBool());
    return {gq, gk, {}, {}};
  }
};

std::pair<Tensor, std::optional<Tensor>> axial_rotary(const Tensor& q, const std::optional<Tensor>& k_opt,
                                                      const Tensor& positions, const std::vector<int64_t>& axes,
                                                      double theta, bool interleaved) {
  const Tensor k = or_undefined(k_opt);
  if (q.dim() != 4) refuse("rotary queries must be (batch, heads, tokens, dim), got ", shape_of(q));
  if (k.defined() && k.dim() != 4) refuse("rotary keys must be (batch, heads, tokens, dim), got ", shape_of(k));
  const int64_t b = q.size(0), t = q.size(2), d = q.size(3), n = static_cast<int64_t>(axes.size());
  if (k.defined() && (k.scalar_type() != q.scalar_type() || k.size(0) != b || k.size(2) != t || k.size(3) != d))
    refuse("queries ", shape_of(q), " ", q.scalar_type(), " and keys ", shape_of(k), " ", k.scalar_type(),
           " do not match");
  RotaryHow how{{}, theta, interleaved};
  int64_t sum = 0;
  bool fine = n > 0;
  for (int64_t w : axes) {
    fine = fine && w > 0 && w % 2 == 0 && w <= d;
    sum += w;
    how.widths.push_back(static_cast<int32_t>(w));
  }
  if (!fine || sum > d)
    refuse("axis widths must be positive, even and sum to at most the head dimension ", d);
  const bool whole = positions.dim() == 2 && positions.size(0) == t && positions.size(1) == n;
  const bool each = positions.dim() == 3 && positions.size(0) == b && positions.size(1) == t && positions.size(2) == n;
  if (!whole && !each)
    refuse("positions must be (", t, ", ", n, ") or (", b, ", ", t, ", ", n, "), got ", shape_of(positions));
  dtype_code(q.scalar_type());
  no_tangents("axial_rotary", {&q, &k, &positions});
  require_cuda({&q, &k, &positions});
  Tensor pos = positions.requires_grad() ? positions.detach() : positions;
  if (pos.scalar_type() != at::kFloat || !pos.is_contiguous()) pos = pos.to(at::kFloat).contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k))) {
    const variable_list y = AxialRotary::apply(q, k_opt, pos, how);
    return {y[0], y.size() > 1 ? std::optional<Tensor>(y[1]) : std::nullopt};
  }
  const auto [yq, yk] = turn(q, k, pos, how, false, false);
  return {yq, yk.defined() ? std::optional<Tensor>(yk) : std::nullopt};
}

// --- layer norm ---------------------------------------------------------------

// weight and bias: vectors that follow one another at the same stride, one for
// each segment of the rows (either may be undefined; run_norm sees to it).
struct NormHow {
  int64_t segments;
  bool add_one;
  double eps;
};

int vector_dtype(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  return dtype_code((weight.defined() ? weight : bias.defined() ? bias : x).scalar_type());
}

int64_t vector_stride(const Tensor& v, const NormHow& how, int64_t features) {
  return how.segments == 1 || !v.defined() ? features : v.stride(0);
}

Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const NormHow& how, Tensor* stats) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int64_t features = x.size(-1), rows = x.numel() / features;
  const Tensor y = at::empty_like(x);
  float* mean = nullptr;
  if (stats) {
    *stats = at::empty({2 * rows}, x.options().dtype(at::kFloat));
    mean = rows ? static_cast<float*>(stats->data_ptr()) : nullptr;
  }
  check(convrot_layer_norm(x.data_ptr(), dtype_code(x.scalar_type()), rows, features, address(weight), address(bias),
                           vector_dtype(x, weight, bias), std::max<int64_t>(1, rows / how.segments),
                           vector_stride(weight.defined() ? weight : bias, how, features), how.add_one,
                           static_cast<float>(how.eps), y.data_ptr(), mean, mean ? mean + rows : nullptr, stream_of(x)),
        "convrot_layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, const NormHow& how) {
    Tensor stats;
    const Tensor w = or_undefined(weight), b = or_undefined(bias);
    const Tensor y = norm_forward(x, w, b, how, &stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["segments"] = how.segments;
    ctx->saved_data["add_one"] = how.add_one;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3];
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const NormHow how{ctx->saved_data["segments"].toInt(), ctx->saved_data["add_one"].toBool(), 0.0};
    const Tensor dy = grads[0].contiguous();
    const int64_t features = x.size(-1), rows = x.numel() / features, per = std::max<int64_t>(1, rows / how.segments);
    const Tensor dx = at::empty_like(x);
    auto sums_like = [&](const Tensor& v) {
      return rows ? at::empty(v.sizes(), v.options()) : at::zeros(v.sizes(), v.options());
    };
    // edges are counted over the tensors that were given
    size_t edge = 1;
    Tensor dw, db, space;
    if (weight.defined() && ctx->needs_input_grad(edge++)) dw = sums_like(weight);
    if (bias.defined() && ctx->needs_input_grad(edge)) db = sums_like(bias);
    int64_t size = 0;
    if (dw.defined() || db.defined()) {
      size = convrot_layer_norm_workspace(rows, features, per);
      space = at::empty({size}, x.options().dtype(at::kByte));
    }
    const auto* mean = static_cast<const float*>(stats.data_ptr());
    check(convrot_layer_norm_backward(x.data_ptr(), dy.data_ptr(), dtype_code(x.scalar_type()), rows, features,
                                      address(weight), vector_dtype(x, weight, bias), per,
                                      vector_stride(weight, how, features), how.add_one, mean, mean + rows,
                                      dx.data_ptr(), address(dw), address(db), address(space), size, stream_of(x)),
          "convrot_layer_norm_backward");
    return {dx, dw, db, {}};
  }
};

Tensor run_norm(Tensor x, Tensor weight, Tensor bias, const NormHow& how) {
  if (!(how.eps >= 0)) refuse("eps must be non-negative, got ", how.eps);
  dtype_code(x.scalar_type());
  no_tangents(how.add_one ? "modulated_layer_norm" : "layer_norm", {&x, &weight, &bias});
  require_cuda({&x, &weight, &bias});
  // both vectors of x's dtype, or both float32
  for (const Tensor* t : {&weight, &bias}) {
    const Tensor& other = t == &weight ? bias : weight;
    if (t->defined() && ((t->scalar_type() != x.scalar_type() && t->scalar_type() != at::kFloat) ||
                         (other.defined() && other.scalar_type() != t->scalar_type()))) {
      weight = weight.defined() ? weight.to(at::kFloat) : weight;
      bias = bias.defined() ? bias.to(at::kFloat) : bias;
      break;
    }
  }
  // After the conversion, which packs the one vector that it touches: unit
  // stride, and segments at one stride that covers the features.
  auto inner = [](const Tensor& t) { return !t.defined() || t.stride(-1) == 1; };
  const bool split = how.segments > 1 && weight.defined() && bias.defined() &&
                     (weight.stride(0) != bias.stride(0) || weight.stride(0) < x.size(-1));
  if (!inner(weight) || !inner(bias) || split) {
    weight = weight.defined() ? weight.contiguous() : weight;
    bias = bias.defined() ? bias.contiguous() : bias;
  }
  if (!x.is_contiguous()) x = x.contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNorm::apply(x, weight.defined() ? std::optional<Tensor>(weight) : std::nullopt,
                            bias.defined() ? std::optional<Tensor>(bias) : std::nullopt, how);
  return norm_forward(x, weight, bias, how, nullptr);
}

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  if (x.dim() == 0 || x.size(-1) == 0)
    refuse("layer norm expects features in the last dimension, got ", shape_of(x));
  const int64_t features = x.size(-1);
  Tensor v[2] = {or_undefined(weight), or_undefined(bias)};
  for (int i = 0; i < 2; ++i) {
    if (!v[i].defined()) continue;
    if (v[i].dim() != 1 || v[i].size(0) != features)
      refuse("layer norm ", i ? "bias" : "weight", " must have shape (", features, ",), got ", shape_of(v[i]));
  }
  return run_norm(x, v[0], v[1], {1, false, eps});
}

Tensor modulated_layer_norm(const Tensor& x, Tensor shift, Tensor scale, double eps) {
  if (x.dim() < 2 || x.size(-1) == 0)
    refuse("modulated layer norm expects (batch, ..., features), got ", shape_of(x));
  const int64_t batch = x.size(0), features = x.size(-1);
  for (const Tensor* v : {&shift, &scale}) {
    const bool fits = (v->dim() == 2 || (v->dim() == 3 && v->size(1) == 1)) && v->size(-1) == features &&
                      (v->size(0) == batch || v->size(0) == 1);
    if (!fits)
      refuse("modulation vector of shape ", shape_of(*v), " does not match (", batch, ", 1, ", features, ")");
  }
  if (shift.size(0) != scale.size(0)) {  // the shared one is repeated, its gradient summed over the samples
    shift = shift.reshape({-1, features}).expand({batch, features});
    scale = scale.reshape({-1, features}).expand({batch, features});
  }
  return run_norm(x, scale, shift, {std::max<int64_t>(1, scale.size(0)), true, eps});
}

// --- GELU with its input saved in 8 bits -----------------------------------------

// Codes, then from the next multiple of 16 bytes on the scales: one allocation.
struct Saved {
  int64_t rows, features, scales_at, bytes;
  Saved(int64_t rows, int64_t features)
      : rows(rows),
        features(features),
        scales_at((rows * features + 15) / 16 * 16),
        bytes(scales_at + 4 * rows * ((features + kSavedGroup - 1) / kSavedGroup)) {}
};

Tensor gelu_forward(const Tensor& x, Tensor* saved) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int64_t features = x.size(-1), rows = x.numel() / features;
  const Tensor y = at::empty_like(x);
  int8_t* codes = nullptr;
  float* scales = nullptr;
  if (saved && rows > 0) {
    const Saved layout(rows, features);
    *saved = at::empty({layout.bytes}, x.options().dtype(at::kChar));
    codes = static_cast<int8_t*>(saved->data_ptr());
    scales = reinterpret_cast<float*>(codes + layout.scales_at);
  }
  check(convrot_gelu_saved8(x.data_ptr(), dtype_code(x.scalar_type()), rows, features, y.data_ptr(), codes, scales,
                            stream_of(x)),
        "convrot_gelu_saved8");
  return y;
}

struct GeluSaved8 : torch::autograd::Function<GeluSaved8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x) {
    Tensor saved;
    const Tensor y = gelu_forward(x, &saved);
    ctx->save_for_backward({saved});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gelu_tanh_saved8");
    const Tensor dy = grads[0].contiguous();
    const c10::cuda::OptionalCUDAGuard guard(dy.device());
    const Tensor dx = at::empty_like(dy);
    const int64_t features = dy.size(-1), rows = dy.numel() / features;
    if (rows == 0) return {dx};
    const Tensor saved = ctx->get_saved_variables()[0];
    const auto* codes = static_cast<const int8_t*>(saved.data_ptr());
    const auto* scales = reinterpret_cast<const float*>(codes + Saved(rows, features).scales_at);
    check(convrot_gelu_saved8_backward(dy.data_ptr(), dtype_code(dy.scalar_type()), rows, features, codes, scales,
                                       dx.data_ptr(), stream_of(dy)),
          "convrot_gelu_saved8_backward");
    return {dx};
  }
};

Tensor gelu_tanh_saved8(Tensor x) {
  if (x.dim() == 0 || x.size(-1) == 0) refuse("gelu expects features in the last dimension, got ", shape_of(x));
  dtype_code(x.scalar_type());
  no_tangents("gelu_tanh_saved8", {&x});
  require_cuda({&x});
  if (!x.is_contiguous()) x = x.contiguous();
  if (at::GradMode::is_enabled() && x.requires_grad()) return GeluSaved8::apply(x);
  return gelu_forward(x, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("int8_linear", &int8_linear);
  m.def("axial_rotary", &axial_rotary);
  m.def("layer_norm", &layer_norm);
  m.def("modulated_layer_norm", &modulated_layer_norm);
  m.def("gelu_tanh_saved8", &gelu_tanh_saved8);
}
