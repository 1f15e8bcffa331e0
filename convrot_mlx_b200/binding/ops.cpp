// Torch-side entry points of the 8-bit and training operators: argument
// checks, output allocation, autograd nodes and the call of the C ABI
// (include/convrot_b200.h), in C++ so that a small call is not bound by the
// interpreter and a backward pass needs no interpreter at all.  The Python
// modules int8, rotary, norm and activation hold the public functions and
// their documentation; everything they refuse is refused here.
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/python_variable.h>

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
    const Tensor qweight = padded_rows(saved[0]), wscales = saved[1].contiguous();  // hooks may have packed the rows
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

// --- 8-bit floating-point linear ------------------------------------------------

constexpr int64_t kSpan = 128;  // values of a row, rows and columns of a weight, that share a scale

// The quantizer and the product in one call; n columns out.
Tensor fp8_product(const Tensor& x, const Tensor& qweight, int layout, const Tensor& wscales, const Tensor& bias,
                   int64_t n) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const Tensor r = rows_of(x);
  const int64_t m = r.size(0), k = r.size(1), pitch = (k + kPitch - 1) / kPitch * kPitch;
  const int64_t scales_pitch = (k + 4 * kSpan - 1) / (4 * kSpan) * 4;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  const Tensor out = at::empty(shape, x.options());
  const Tensor space = at::empty({m * (pitch + scales_pitch)}, x.options().dtype(at::kByte));  // codes, then scales
  auto* codes = static_cast<uint8_t*>(space.data_ptr());
  uint8_t* scales = codes + m * pitch;
  const int dtype = dtype_code(x.scalar_type());
  const auto* weight = static_cast<const uint8_t*>(qweight.data_ptr());
  const auto* ws = static_cast<const uint8_t*>(wscales.data_ptr());
  const auto* b = static_cast<const float*>(address(bias));
  check(convrot_fp8_linear(r.data_ptr(), dtype, r.stride(0), weight, qweight.stride(0), layout, ws, wscales.size(1), b,
                           out.data_ptr(), dtype, m, n, k, codes, pitch, scales, scales_pitch, stream_of(x)),
        "convrot_fp8_linear");
  return out;
}

// padded_rows, and the last row too can be read in whole 16 bytes.
Tensor whole_rows(const Tensor& codes) {
  const Tensor t = padded_rows(codes);
  const int64_t last = (t.size(0) - 1) * t.stride(0) + (t.size(1) + kPitch - 1) / kPitch * kPitch;
  if (static_cast<int64_t>(t.storage().nbytes()) >= t.storage_offset() + last) return t;
  const Tensor rows = at::empty({t.size(0), (t.size(1) + kPitch - 1) / kPitch * kPitch}, t.options());
  const Tensor out = rows.narrow(1, 0, t.size(1));
  out.copy_(t);
  return out;
}

// The gradient of the input; a node of its own, which costs a small call less
// than torch::autograd::Function.
struct Fp8LinearBackward : torch::autograd::Node {
  torch::autograd::SavedVariable qweight, wscales;
  variable_list apply(variable_list&& grads) override {
    once("fp8_linear");
    const std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {Tensor()};
    // hooks of saved tensors may have packed the rows
    const Tensor w = whole_rows(qweight.unpack()), ws = wscales.unpack().contiguous();
    return {fp8_product(grads[0], w, CONVROT_LAYOUT_KN, ws, {}, w.size(1))};
  }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    qweight.reset_data();
    wscales.reset_data();
  }
  std::string name() const override { return "Fp8LinearBackward"; }
};

Tensor fp8_linear(const Tensor& x, const Tensor& qweight, const Tensor& wscales, const std::optional<Tensor>& bias) {
  if (x.dim() == 0) refuse("fp8 linear expects at least one dimension");
  if (qweight.dim() != 2 || qweight.scalar_type() != at::kFloat8_e4m3fn)
    refuse("fp8 weight must be a 2D float8_e4m3fn tensor, got ", shape_of(qweight), " ", qweight.scalar_type());
  const int64_t n = qweight.size(0), k = x.size(-1);
  if (qweight.size(1) != k || k == 0 || n == 0)
    refuse("fp8 weight must be (N, K) rows; activation K=", k, ", weight=", shape_of(qweight));
  const int64_t nb = (n + kSpan - 1) / kSpan, kb = (k + kSpan - 1) / kSpan;
  if (wscales.dim() != 2 || wscales.size(0) != nb || wscales.size(1) != kb || wscales.scalar_type() != at::kFloat8_e8m0fnu)
    refuse("fp8 weight scales must be (", nb, ", ", kb, ") float8_e8m0fnu, got ", shape_of(wscales), " ",
           wscales.scalar_type());
  const Tensor b = or_undefined(bias);
  if (b.defined() && (b.dim() != 1 || b.size(0) != n))
    refuse("fp8 bias must have shape (", n, ",), got ", shape_of(b));
  if (wants_grad(qweight) || wants_grad(wscales) || wants_grad(b))
    refuse("the weight, its scales and the bias of an fp8 linear are frozen: they may not require gradients");
  dtype_code(x.scalar_type());
  no_tangents("fp8_linear", {&x, &b});
  require_cuda({&x, &qweight, &wscales, &b});
  const Tensor w = whole_rows(qweight), ws = wscales.contiguous(), fb = f32_vector(b);
  if (!at::GradMode::is_enabled() || !x.requires_grad()) return fp8_product(x, w, CONVROT_LAYOUT_NK, ws, fb, n);
  const std::shared_ptr<Fp8LinearBackward> node(new Fp8LinearBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  node->qweight = torch::autograd::SavedVariable(w, /*is_output=*/false);
  node->wscales = torch::autograd::SavedVariable(ws, /*is_output=*/false);
  Tensor y;
  {
    const at::NoGradGuard no_grad;
    y = fp8_product(x, w, CONVROT_LAYOUT_NK, ws, fb, n);
  }
  torch::autograd::set_history(y, node);
  return y;
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
    const auto [gq, gk] = turn(grads[0], dk, ctx->get_saved_variables()[0].contiguous(), how, true,
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
    // as forward had them, also where hooks of saved tensors have laid them out in another way
    const Tensor x = saved[0].contiguous(), stats = saved[3].contiguous();
    Tensor weight = saved[1];
    const Tensor& bias = saved[2];
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const NormHow how{ctx->saved_data["segments"].toInt(), ctx->saved_data["add_one"].toBool(), 0.0};
    if (weight.defined() && (weight.stride(-1) != 1 || (how.segments > 1 && weight.stride(0) < x.size(-1))))
      weight = weight.contiguous();
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
    Tensor saved = ctx->get_saved_variables()[0].contiguous();
    if (reinterpret_cast<uintptr_t>(saved.data_ptr()) % 16) saved = saved.clone();  // its scales are float32
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

// --- AdamW and the gradient norm ---------------------------------------------------

// The tensors of a Python sequence without a reference each (the caller holds
// the sequence for the length of the call); nothing where it has None.
class TensorList {
 public:
  TensorList(const py::object& o, const char* what) : what_(what) {
    seq_ = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "expected a sequence of tensors"));
    if (!seq_) throw py::error_already_set();
    items_ = PySequence_Fast_ITEMS(seq_.ptr());
    size_ = PySequence_Fast_GET_SIZE(seq_.ptr());
  }
  int64_t size() const { return size_; }
  const Tensor* at(int64_t i) const {
    if (items_[i] == Py_None) return nullptr;
    if (!THPVariable_Check(items_[i])) refuse(what_, " must be tensors, got ", Py_TYPE(items_[i])->tp_name);
    return &THPVariable_Unpack(items_[i]);
  }

 private:
  py::object seq_;
  PyObject** items_;
  int64_t size_;
  const char* what_;
};

int dtype_slot(const Tensor& t) { return dtype_code(t.scalar_type()); }  // 0, 1 or 2

// t where its values are dense in memory in some order, else packed.
Tensor dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense() ? t : t.contiguous(); }

// Gradients of one device as the sums of squares take them, by type.
struct GradLists {
  std::vector<convrot_grad_tensor> by_type[3];
  std::vector<Tensor> held;
  c10::Device home;

  explicit GradLists(const std::vector<const Tensor*>& grads) : home(grads.front()->device()) {
    require_cuda({grads.front()});
    for (const Tensor* g : grads) {
      if (g->layout() != at::kStrided) refuse("gradients must be dense tensors");
      if (g->device() != home) refuse("expected all tensors on ", home.str(), ", got one on ", g->device().str());
      const Tensor* t = g;
      if (!g->is_contiguous()) {
        held.push_back(dense(*g));
        t = &held.back();
      }
      by_type[dtype_slot(*g)].push_back({t->data_ptr(), t->numel()});
    }
  }
  int64_t count(int type) const { return static_cast<int64_t>(by_type[type].size()); }
};

// Partial sums of the squares of gradients of any of the three types in one
// tensor.
Tensor sums_of(const GradLists& lists, const Tensor& like) {
  const c10::cuda::OptionalCUDAGuard guard(lists.home);
  int64_t counts[3] = {}, total = 0;
  for (int i = 0; i < 3; ++i)
    if (lists.count(i)) total += counts[i] = convrot_square_sums_count(lists.count(i), lists.by_type[i].data());
  const Tensor sums = at::empty({total}, like.options().dtype(at::kDouble).requires_grad(false));
  auto* at = static_cast<double*>(sums.data_ptr());
  for (int i = 0; i < 3; ++i) {
    if (!counts[i]) continue;
    check(convrot_square_sums(lists.count(i), lists.by_type[i].data(), i, at, counts[i], nullptr, stream_of(like)),
          "convrot_square_sums");
    at += counts[i];
  }
  return sums;
}
Tensor square_sums_of(const std::vector<const Tensor*>& grads) { return sums_of(GradLists(grads), *grads.front()); }

void write_norm(const Tensor& sums, float* to) {
  check(convrot_norm_of_sums(static_cast<const double*>(sums.data_ptr()), sums.numel(), to, stream_of(sums)),
        "convrot_norm_of_sums");
}
Tensor norm_of(const Tensor& sums) {
  const c10::cuda::OptionalCUDAGuard guard(sums.device());
  const Tensor norm = at::empty({}, sums.options().dtype(at::kFloat));
  write_norm(sums, static_cast<float*>(norm.data_ptr()));
  return norm;
}

std::vector<const Tensor*> present(const TensorList& list) {
  std::vector<const Tensor*> out;
  out.reserve(list.size());
  for (int64_t i = 0; i < list.size(); ++i)
    if (const Tensor* t = list.at(i)) out.push_back(t);
  if (out.empty()) refuse("expected at least one gradient");
  return out;
}

Tensor square_sums(const py::object& grads) {
  const at::NoGradGuard no_grad;
  const TensorList list(grads, "gradients");
  return square_sums_of(present(list));
}

// Chunks of 2048 values whose norm is one launch's: 8 CTAs with 16 each.
constexpr int64_t kOneLaunch = 128;

Tensor grad_norm(const py::object& grads) {
  const at::NoGradGuard no_grad;
  const TensorList list(grads, "gradients");
  const std::vector<const Tensor*> tensors = present(list);
  const GradLists lists(tensors);
  const Tensor& first = *tensors.front();
  const c10::cuda::OptionalCUDAGuard guard(lists.home);
  const Tensor norm = at::empty({}, first.options().dtype(at::kFloat).requires_grad(false));
  auto* to = static_cast<float*>(norm.data_ptr());
  const int type = dtype_slot(first);
  if (lists.count(type) == static_cast<int64_t>(tensors.size()) && lists.count(type) <= 1024) {
    int64_t chunks = 0;
    for (const convrot_grad_tensor& t : lists.by_type[type]) chunks += (t.numel + 2047) / 2048;
    if (chunks <= kOneLaunch) {
      check(convrot_square_sums(lists.count(type), lists.by_type[type].data(), type, nullptr,
                                std::max<int64_t>(1, std::min<int64_t>(8, (chunks + 3) / 4)), to, stream_of(first)),
            "convrot_square_sums");
      return norm;
    }
  }
  write_norm(sums_of(lists, first), to);
  return norm;
}

// Whether the values of two tensors of one shape lie in memory in the same
// order, both without gaps if one is.
bool same_layout(const Tensor& a, const Tensor& b) {
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// A scalar that is a number, or one float32 on the device.
const float* device_scalar(const py::object& o, const char* what, const c10::Device& home, double* number) {
  if (!THPVariable_Check(o.ptr())) {
    *number = o.cast<double>();
    return nullptr;
  }
  const Tensor& t = THPVariable_Unpack(o.ptr());
  if (t.numel() != 1 || t.scalar_type() != at::kFloat || t.device() != home)
    refuse("a ", what, " on the device must be one float32 on ", home.str());
  return static_cast<const float*>(t.data_ptr());
}

// The tensors of a step in memory: a parameter's gradient may be itself (or its
// moments), whose values are read before they are written, and two parameters
// may have one gradient, but nothing that is written may overlap anything else.
class Spans {
 public:
  enum Kind { kParam, kMoment, kRoot, kScales, kGrad, kKinds };

  explicit Spans(int64_t count) { storages_.reserve(kKinds * count); }

  // A tensor whose values are dense in memory; a parameter's own tensors after it.
  void add(Kind kind, const Tensor& t, const void* at, int64_t bytes) {
    const auto start = reinterpret_cast<uintptr_t>(at);
    Range& range = ranges_[kind];
    range.ascending &= start >= range.end;
    if (!range.end) range.first = start;
    range.end = start + bytes;
    // the lowest bit: only read
    storages_.push_back(reinterpret_cast<uintptr_t>(t.unsafeGetTensorImpl()->unsafe_storage().data()) & ~uintptr_t(1) |
                        (kind == kGrad));
  }

  // by_type: the same tensors.
  bool disjoint(const std::vector<convrot_adamw_tensor> (&by_type)[3], bool eight) const {
    return in_order() || in_storages_of_their_own() || swept(by_type, eight);
  }

 private:
  struct Range {
    uintptr_t first = 0, end = 0;
    bool ascending = true;
  };
  struct Span {
    uintptr_t at, end;
    int64_t index;  // of the parameter
  };

  // Each kind in a stretch of memory of its own, one tensor after another: packed buffers.
  bool in_order() const {
    for (int i = 0; i < kKinds; ++i) {
      if (!ranges_[i].ascending) return false;
      for (int j = 0; j < i; ++j)
        if (ranges_[i].first < ranges_[j].end && ranges_[j].first < ranges_[i].end) return false;
    }
    return true;
  }

  // Tensors allocated one by one, whatever their order.
  bool in_storages_of_their_own() const {
    size_t size = 64;
    while (2 * size < 3 * storages_.size()) size *= 2;
    std::vector<uintptr_t> table(size, 0);
    for (const uintptr_t storage : storages_) {
      const uintptr_t base = storage & ~uintptr_t(1);
      size_t i = (base >> 4) * 0x9E3779B97F4A7C15ull >> 20 & (size - 1);
      for (; table[i]; i = (i + 1) & (size - 1))
        if ((table[i] & ~uintptr_t(1)) == base && !(table[i] & storage & 1)) return false;
      table[i] = storage;
    }
    return true;
  }

  // In the order of their starts, what is written first: spans that are written
  // may not overlap, so the last of them is the only one that reaches on.
  static bool swept(const std::vector<convrot_adamw_tensor> (&by_type)[3], bool eight) {
    std::vector<Span> spans[kKinds];
    int64_t index = 0;
    for (int type = 0; type < 3; ++type) {
      const int64_t e = type == CONVROT_F32 ? 4 : 2, moment = eight ? 1 : 4;
      for (const convrot_adamw_tensor& t : by_type[type]) {
        auto add = [&](Kind kind, const void* at, int64_t bytes) {
          const auto start = reinterpret_cast<uintptr_t>(at);
          spans[kind].push_back({start, start + bytes, index});
        };
        add(kParam, t.param, e * t.numel);
        add(kMoment, t.exp_avg, moment * t.numel);
        add(kRoot, t.exp_avg_sq, moment * t.numel);
        if (eight) add(kScales, t.scales, (t.numel + 255) / 256 * 8);
        add(kGrad, t.grad, e * t.numel);
        ++index;
      }
    }
    for (auto& list : spans) std::sort(list.begin(), list.end(), [](const Span& a, const Span& b) { return a.at < b.at; });
    size_t next[kKinds] = {};
    Span written{0, 0, -1};
    uintptr_t read_end = 0;
    for (;;) {
      int kind = -1;
      for (int k = 0; k < kKinds; ++k)
        if (next[k] < spans[k].size() && (kind < 0 || spans[k][next[k]].at < spans[kind][next[kind]].at)) kind = k;
      if (kind < 0) return true;
      const Span& s = spans[kind][next[kind]++];
      if (kind == kGrad) {
        const bool own = s.index == written.index && s.at == written.at && s.end == written.end;
        if (s.at < written.end && !own) return false;
        read_end = std::max(read_end, s.end);
      } else {
        if (s.at < written.end || s.at < read_end) return false;
        written = s;
      }
    }
  }

  std::vector<uintptr_t> storages_;
  Range ranges_[kKinds];
};

// The step; with max_norm the gradients' norm, else nothing.  sums: of
// square_sums, where the norm is over more gradients than these.
std::optional<Tensor> adamw_step(const py::object& params, const py::object& grads, const py::object& exp_avgs,
                                 const py::object& exp_avg_sqs, const py::object& scales, const py::object& step,
                                 const py::object& lr, double beta1, double beta2, double eps, double weight_decay,
                                 std::optional<double> max_norm, const std::optional<Tensor>& sums_in) {
  const at::NoGradGuard no_grad;
  const TensorList p(params, "parameters"), g(grads, "gradients"), m(exp_avgs, "moments"), v(exp_avg_sqs, "moments");
  const bool eight = !scales.is_none();
  const TensorList s(eight ? scales : exp_avgs, "scales");
  const int64_t count = p.size();
  if (g.size() != count || m.size() != count || v.size() != count || s.size() != count)
    refuse("parameters, gradients, moments and scales must be equally many, got ", count, ", ", g.size(), ", ", m.size(),
           ", ", v.size(), " and ", s.size());
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) refuse("betas must be in [0, 1), got ", beta1, " and ", beta2);
  if (!(eps >= 0) || !(weight_decay >= 0)) refuse("eps and weight decay must be non-negative");
  if (max_norm && !(*max_norm >= 0)) refuse("the largest norm must be non-negative, got ", *max_norm);
  const at::ScalarType moment = eight ? at::kFloat8_e4m3fn : at::kFloat;
  std::vector<convrot_adamw_tensor> by_type[3];
  std::vector<const Tensor*> used, written;
  const Tensor* given = nullptr;  // a gradient, with values or without
  std::vector<Tensor> held;
  Spans spans(count);
  for (auto& list : by_type) list.reserve(count);
  used.reserve(count);
  written.reserve(4 * count);
  c10::Device home(c10::DeviceType::CPU);
  for (int64_t i = 0; i < count; ++i) {
    const Tensor* gi = g.at(i);
    if (!gi) continue;
    given = gi;
    const Tensor *pi = p.at(i), *mi = m.at(i), *vi = v.at(i), *si = eight ? s.at(i) : mi;
    if (!pi || !mi || !vi || !si) refuse("parameter ", i, " has a gradient, but a parameter, moment or scale is missing");
    if (used.empty()) home = pi->device();
    for (const Tensor* t : {pi, gi, mi, vi, si}) {
      const c10::Device at = t->device();
      if (!at.is_cuda() || at != home) require_cuda({used.empty() ? pi : written.front(), t});
      if (t->layout() != at::kStrided) refuse("the AdamW step takes dense tensors");
    }
    if (gi->scalar_type() != pi->scalar_type() || gi->sizes() != pi->sizes())
      refuse("gradient ", i, " is ", shape_of(*gi), " ", gi->scalar_type(), ", its parameter ", shape_of(*pi), " ",
             pi->scalar_type());
    for (const Tensor* t : {mi, vi})
      if (t->scalar_type() != moment || t->sizes() != pi->sizes())
        refuse("moments of parameter ", i, " must be ", shape_of(*pi), " ", moment, ", got ", shape_of(*t), " ",
               t->scalar_type());
    const int64_t n = pi->numel(), blocks = (n + 255) / 256;
    if (eight && (si->scalar_type() != at::kFloat || si->dim() != 2 || si->size(0) != blocks || si->size(1) != 2 ||
                  !si->is_contiguous()))
      refuse("scales of parameter ", i, " must be (", blocks, ", 2) float32 and contiguous, got ", shape_of(*si), " ",
             si->scalar_type());
    const Tensor* grad = gi;
    if (!pi->is_contiguous() || !mi->is_contiguous() || !vi->is_contiguous() || !gi->is_contiguous()) {
      // values are taken in memory order: one order for all four
      if (!pi->is_non_overlapping_and_dense() || !same_layout(*mi, *pi) || !same_layout(*vi, *pi))
        refuse("parameter ", i, " must be dense in memory, and its moments laid out as it is");
      if (!same_layout(*gi, *pi)) {
        held.push_back(at::empty_strided(pi->sizes(), pi->strides(), gi->options()).copy_(gi->detach()));
        grad = &held.back();
      }
    }
    if (n == 0) continue;
    void *const p_at = pi->data_ptr(), *const m_at = mi->data_ptr(), *const v_at = vi->data_ptr();
    const void* g_at = grad->const_data_ptr();
    auto* s_at = eight ? static_cast<float*>(si->data_ptr()) : nullptr;
    by_type[dtype_slot(*pi)].push_back({p_at, g_at, m_at, v_at, s_at, n});
    const int64_t bytes = n * pi->element_size(), moment_bytes = n * (eight ? 1 : 4);
    spans.add(Spans::kParam, *pi, p_at, bytes);
    spans.add(Spans::kMoment, *mi, m_at, moment_bytes);
    spans.add(Spans::kRoot, *vi, v_at, moment_bytes);
    if (eight) spans.add(Spans::kScales, *si, s_at, 8 * blocks);
    spans.add(Spans::kGrad, *grad, g_at, bytes);
    used.push_back(gi);
    written.insert(written.end(), {pi, mi, vi});
    if (eight) written.push_back(si);
  }
  if (!spans.disjoint(by_type, eight))
    refuse("a parameter, a moment or its scales overlaps another tensor of the step (or occurs twice)");
  convrot_adamw_options o = {};
  if (used.empty()) {
    if (!max_norm) return std::nullopt;
    if (!given) refuse("clipping needs at least one gradient");
    if (sums_in.has_value()) return norm_of(*sums_in);
    return at::zeros({}, given->options().dtype(at::kFloat).requires_grad(false));  // of no values
  }
  o.step_device = device_scalar(step, "step", home, &o.step);
  o.lr_device = device_scalar(lr, "learning rate", home, &o.lr);
  if (!o.step_device && !(o.step >= 1)) refuse("the step counts from 1, got ", o.step);
  if (!o.lr_device && !(o.lr >= 0)) refuse("the learning rate must be non-negative, got ", o.lr);
  o.beta1 = beta1, o.beta2 = beta2, o.eps = eps, o.weight_decay = weight_decay;
  const c10::cuda::OptionalCUDAGuard guard(home);
  std::optional<Tensor> norm;
  Tensor sums;
  if (max_norm) {
    sums = sums_in.has_value() ? *sums_in : square_sums_of(used);
    if (sums.scalar_type() != at::kDouble || sums.device() != home || !sums.is_contiguous() || sums.numel() == 0)
      refuse("sums of squares must be float64 on ", home.str());
    norm = at::empty({}, sums.options().dtype(at::kFloat));
    o.sums = static_cast<const double*>(sums.data_ptr());
    o.sums_count = sums.numel();
    o.max_norm = *max_norm;
    o.norm = static_cast<float*>(norm->data_ptr());
  }
  for (int i = 0; i < 3; ++i) {
    if (by_type[i].empty()) continue;
    check(convrot_adamw(static_cast<int64_t>(by_type[i].size()), by_type[i].data(), i, eight ? 8 : 32, &o,
                        stream_of(*written.front())),
          "convrot_adamw");
  }
  for (const Tensor* t : written)  // autograd is to see it
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("int8_linear", &int8_linear);
  m.def("fp8_linear", &fp8_linear);
  m.def("square_sums", &square_sums);
  m.def("grad_norm", &grad_norm);
  m.def("adamw_step", &adamw_step);
  m.def("axial_rotary", &axial_rotary);
  m.def("layer_norm", &layer_norm);
  m.def("modulated_layer_norm", &modulated_layer_norm);
  m.def("gelu_tanh_saved8", &gelu_tanh_saved8);
}
