// flb_ops: the row operators' torch side in C++: argument checks, buffers, streams, devices and autograd
// functions around the C ABI of libflb_b200.so. In C++ because a training step through a small row operator
// is bound by the host: as Python functions, forward and backward of a norm over 192 rows took 146 us on a B200
// machine, nearly all of it the interpreter's. The Python packages keep the operators' names, their
// documentation and their torch.func rules. There is no CPU path.
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "flb_b200.h"

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;

int dtype_of(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return FLB_F32;
    case at::kHalf: return FLB_F16;
    case at::kBFloat16: return FLB_BF16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, float16 or bfloat16, not ", t);
  }
}
int dtype_of(const Tensor& t, const char* name) { return dtype_of(t.scalar_type(), name); }

void need_cuda(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "flb-transformer_b200 runs on CUDA tensors only (sm_100a kernels; no CPU path); got a tensor on ",
              t.device());
}
void same_device(const Tensor& x, const Opt& t) {
  if (!t || !t->defined()) return;
  need_cuda(*t);
  TORCH_CHECK_VALUE(t->device() == x.device(), "tensors on different devices: ", x.device(), " and ", t->device());
}
bool given(const Opt& t) { return t && t->defined(); }

// The operators have no forward-mode derivative: an input with a tangent would lose it without a word. (A tangent does not set
// requires_grad.)
void no_tangent(const Opt& t, const char* what) {
  TORCH_CHECK(!given(t) || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t->_fw_grad(0).defined(), what,
              " has no forward-mode derivative");
}
void* ptr(const Opt& t) { return given(t) ? t->data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void check(int st, const char* what) {
  static const char* const names[] = {"OK", "SHAPE", "DTYPE", "ALIGN", "TIMEOUT", "LAUNCH", "UNSUPPORTED", "CUDA", "WORKSPACE"};
  TORCH_CHECK(st == FLB_OK, what, " failed with FLB_ERR_", st >= 0 && st < 9 ? names[st] : "?", ": ", flb_last_error());
}
Tensor buffer(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

// x's leading axes as one axis of rows, a fixed number of elements apart: x itself where its strides allow
// it, else a contiguous copy.
std::tuple<Tensor, int64_t> rows_of(const Tensor& x) {
  const int64_t D = x.size(-1);
  if (x.is_contiguous()) return {x, D};
  if (x.stride(-1) != 1 || x.numel() == 0) return {x.contiguous(), D};
  int64_t pitch = -1, span = 0;
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (pitch < 0) {
      pitch = x.stride(i);
      span = pitch * x.size(i);
    } else if (x.stride(i) == span) {
      span *= x.size(i);
    } else {
      return {x.contiguous(), D};
    }
  }
  return {x, pitch < 0 ? D : pitch};
}

int64_t last_axis(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() >= 1, name, " must have at least one axis");
  return x.size(-1);
}
int64_t rows_in(const Tensor& x) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) n *= x.size(i);
  return n;
}
std::pair<Tensor, Tensor> kept_buffers(int64_t rows, int64_t D, const Tensor& like) {
  return {at::empty({rows, flb_code_pitch(D)}, like.options().dtype(at::kChar)),
          at::empty({rows, flb_kept_blocks(D)}, like.options().dtype(at::kByte))};
}

// The outputs of a backward that was asked for a graph of its own: using that graph raises.
torch::autograd::variable_list differentiable_once(torch::autograd::variable_list out) {
  if (!c10::GradMode::is_enabled()) return out;
  torch::autograd::variable_list in;
  for (auto& t : out)
    if (t.defined()) in.push_back(t.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>("this operator is differentiable once", (int)in.size());
  in = (*error)(std::move(in));
  size_t k = 0;
  for (auto& t : out)
    if (t.defined()) t = in[k++];
  return out;
}

// ---- LayerNorm ----------------------------------------------------------------------------------------

struct NormSizes {
  int dt, wdt;
  int64_t G, R, D;
};

NormSizes check_norm(const Tensor& x, const Opt& weight, const Opt& bias) {
  NormSizes n{dtype_of(x, "x"), 0, 1, 0, 0};
  need_cuda(x);
  same_device(x, weight);
  same_device(x, bias);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last axis of at least one element, not shape ", x.sizes());
  n.D = x.size(-1);
  n.wdt = n.dt;
  const std::pair<const char*, const Opt*> both[] = {{"weight", &weight}, {"bias", &bias}};
  for (auto& [name, t] : both) {
    if (!given(*t)) continue;
    const Tensor& v = **t;
    n.wdt = dtype_of(v, name);
    TORCH_CHECK_TYPE(n.wdt == FLB_F32 || n.wdt == n.dt, name, " must be float32 or ", x.scalar_type(), ", not ", v.scalar_type());
    const bool fits = (v.dim() == 1 || (v.dim() == 2 && x.dim() >= 2 && v.size(0) == x.size(0))) && v.size(-1) == n.D;
    TORCH_CHECK_VALUE(fits, name, " of shape ", v.sizes(), " for x of shape ", x.sizes(), ": [D], or [G, D] with G x's first axis");
    if (v.dim() == 2) n.G = v.size(0);
  }
  if (given(weight) && given(bias))
    TORCH_CHECK_VALUE(weight->sizes() == bias->sizes() && weight->scalar_type() == bias->scalar_type(),
                      "weight and bias differ in shape or type");
  n.R = n.G ? rows_in(x) / n.G : 0;
  return n;
}

Opt contiguous(const Opt& t) { return given(t) ? Opt(t->contiguous()) : Opt(); }

// y, and what the backward reads: (1/sigma, mean, -, -), or with keep8 (1/sigma, -, codes, exps)
std::tuple<Tensor, Opt, Opt, Opt, Opt> norm_forward(const Tensor& x_, const Opt& weight, const Opt& bias, double eps, bool keep8,
                                                    bool stats) {
  const NormSizes n = check_norm(x_, weight, bias);
  TORCH_CHECK(!stats || n.D <= 16384, "layer_norm: the gradient of rows wider than 16384 is not supported");
  const c10::cuda::CUDAGuard guard(x_.device());
  auto [x, ldx] = rows_of(x_);
  const Opt w = contiguous(weight), b = contiguous(bias);
  Tensor y = at::empty(x.sizes(), x.options());
  Opt mean, rstd, codes, exps;
  if (stats) {
    rstd = at::empty({n.G * n.R}, x.options().dtype(at::kFloat));
    if (keep8) std::tie(codes, exps) = kept_buffers(n.G * n.R, n.D, x);
    else mean = at::empty_like(*rstd);
  }
  check(flb_layer_norm_fwd(x.data_ptr(), ldx, ptr(w), ptr(b), n.wdt, y.data_ptr(), (float*)ptr(mean), (float*)ptr(rstd),
                           (int8_t*)ptr(codes), (uint8_t*)ptr(exps), n.G, n.R, n.D, n.dt, (float)eps, stream_of(x)),
        "flb_layer_norm_fwd");
  return {y, rstd, mean, codes, exps};
}

// x and mean, or codes and exps; weight and bias as in the forward (the bias for its shape alone)
std::tuple<Tensor, Opt, Opt> norm_backward(const Opt& x_, const Tensor& rstd, const Opt& mean, const Opt& codes, const Opt& exps,
                                           const Opt& weight, const Opt& bias, const Tensor& dy_, bool want_params) {
  const c10::cuda::CUDAGuard guard(dy_.device());
  const Tensor dy = dy_.contiguous();
  const int64_t D = dy.size(-1), rows = rows_in(dy);
  const int dt = dtype_of(dy, "dy");
  const Opt& like = given(weight) ? weight : bias;
  const int64_t G = given(like) && like->dim() == 2 ? like->size(0) : 1, R = G ? rows / G : 0;
  const int wdt = given(like) ? dtype_of(*like, "weight") : dt;
  Opt x;
  int64_t ldx = D;
  if (given(x_)) {
    auto [t, ld] = rows_of(*x_);
    x = t, ldx = ld;
  }
  const Opt w = contiguous(weight);
  Tensor dx = at::empty_like(dy);
  Opt dw, db;
  Tensor ws;
  size_t need = 0;
  if (given(like) && want_params) {
    dw = at::empty(like->sizes(), like->options());
    db = at::empty(like->sizes(), like->options());
    need = flb_layer_norm_bwd_workspace_bytes(G, R, D);
    if (need) ws = buffer(need, dy);
  }
  check(flb_layer_norm_bwd(ptr(x), ldx, (const int8_t*)ptr(codes), (const uint8_t*)ptr(exps), (const float*)ptr(mean),
                           (const float*)rstd.data_ptr(), ptr(w), wdt, dy.data_ptr(), dx.data_ptr(), ptr(dw), ptr(db), G, R, D, dt,
                           need ? ws.data_ptr() : nullptr, need, stream_of(dy)),
        "flb_layer_norm_bwd");
  return {dx, given(weight) ? dw : Opt(), given(bias) ? db : Opt()};
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Opt& weight, const Opt& bias, double eps,
                        bool keep8) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, rstd, mean, codes, exps] = norm_forward(x, weight, bias, eps, keep8, true);
    auto t = [](const Opt& o) { return given(o) ? *o : Tensor(); };
    ctx->save_for_backward({keep8 ? Tensor() : x, t(rstd), t(mean), t(codes), t(exps), t(weight), t(bias)});
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    const auto s = ctx->get_saved_variables();
    // the places of weight and bias among the inputs that are tensors
    const int at_bias = s[5].defined() ? 2 : 1;
    const bool params = (s[5].defined() && ctx->needs_input_grad(1)) || (s[6].defined() && ctx->needs_input_grad(at_bias));
    torch::autograd::variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dx, dw, db] = norm_backward(s[0], s[1], s[2], s[3], s[4], s[5], s[6], g[0], params);
      out[0] = dx;
      if (dw) out[1] = *dw;
      if (db) out[2] = *db;
    }
    return differentiable_once(std::move(out));
  }
};

bool wants_grad(const Opt& t) { return given(t) && t->requires_grad(); }

Tensor layer_norm(const Tensor& x, const Opt& weight, const Opt& bias, double eps, bool keep8) {
  for (const Opt& t : {Opt(x), weight, bias}) no_tangent(t, "layer_norm");
  if (c10::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias)))
    return LayerNormFn::apply(x, weight, bias, eps, keep8);
  return std::get<0>(norm_forward(x, weight, bias, eps, false, false));
}

// ---- the 8-bit kept form and the gate -------------------------------------------------------------------

std::pair<Tensor, Tensor> pack8(const Tensor& x_) {
  const int dt = dtype_of(x_, "x");
  need_cuda(x_);
  const int64_t D = last_axis(x_, "x"), rows = rows_in(x_);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.contiguous();
  auto [codes, exps] = kept_buffers(rows, D, x);
  if (rows && D)
    check(flb_pack8(x.data_ptr(), (int8_t*)codes.data_ptr(), (uint8_t*)exps.data_ptr(), rows, D, dt, stream_of(x)), "flb_pack8");
  return {codes, exps};
}

Tensor unpack8(const Tensor& codes, const Tensor& exps, std::vector<int64_t> shape, at::ScalarType dtype) {
  const int dt = dtype_of(dtype, "the type");
  TORCH_CHECK_VALUE(!shape.empty(), "a tensor with at least one axis is needed");
  const int64_t D = shape.back();
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar && exps.scalar_type() == at::kByte &&
                        codes.sizes() == at::IntArrayRef({rows, flb_code_pitch(D)}) &&
                        exps.sizes() == at::IntArrayRef({rows, flb_kept_blocks(D)}) && codes.is_contiguous() && exps.is_contiguous(),
                    "codes and exps are not a kept form of shape ", at::IntArrayRef(shape));
  need_cuda(codes);
  same_device(codes, exps);
  const c10::cuda::CUDAGuard guard(codes.device());
  Tensor out = at::empty(shape, codes.options().dtype(dtype));
  if (rows && D)
    check(flb_unpack8((const int8_t*)codes.data_ptr(), (const uint8_t*)exps.data_ptr(), out.data_ptr(), rows, D, dt, stream_of(out)),
          "flb_unpack8");
  return out;
}

// y and, with keep8, the kept forms of x and z
std::vector<Tensor> gate_forward(const Tensor& x_, const Tensor& z_, bool keep8) {
  const int dt = dtype_of(x_, "x");
  need_cuda(x_);
  same_device(x_, z_);
  TORCH_CHECK_VALUE(x_.sizes() == z_.sizes(), "x and z differ in shape: ", x_.sizes(), " ", z_.sizes());
  TORCH_CHECK_TYPE(x_.scalar_type() == z_.scalar_type(), "x and z differ in type: ", x_.scalar_type(), " ", z_.scalar_type());
  const int64_t D = last_axis(x_, "x"), rows = rows_in(x_);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = x_.contiguous(), z = z_.contiguous();
  std::vector<Tensor> out{at::empty_like(x)};
  if (keep8)
    for (int i = 0; i < 2; ++i) {
      auto [c, e] = kept_buffers(rows, D, x);
      out.push_back(c), out.push_back(e);
    }
  auto p = [&](size_t i) { return i < out.size() ? out[i].data_ptr() : nullptr; };
  if (rows && D)
    check(flb_gate_fwd(x.data_ptr(), z.data_ptr(), p(0), (int8_t*)p(1), (uint8_t*)p(2), (int8_t*)p(3), (uint8_t*)p(4), rows, D, dt,
                       stream_of(x)),
          "flb_gate_fwd");
  return out;
}

// kept: x and z, or codes and exps of x and of z
std::pair<Tensor, Tensor> gate_backward(const std::vector<Tensor>& kept, const Tensor& dy_) {
  const c10::cuda::CUDAGuard guard(dy_.device());
  const Tensor dy = dy_.contiguous();
  const int64_t D = dy.size(-1), rows = rows_in(dy);
  Tensor dx = at::empty_like(dy), dz = at::empty_like(dy);
  const bool keep8 = kept.size() == 4;
  Tensor x, z;
  if (!keep8) x = kept[0].contiguous(), z = kept[1].contiguous();
  auto c = [&](int i) { return keep8 ? kept[i].data_ptr() : nullptr; };
  if (rows && D)
    check(flb_gate_bwd(keep8 ? nullptr : x.data_ptr(), keep8 ? nullptr : z.data_ptr(), (const int8_t*)c(0), (const uint8_t*)c(1),
                       (const int8_t*)c(2), (const uint8_t*)c(3), dy.data_ptr(), dx.data_ptr(), dz.data_ptr(), rows, D,
                       dtype_of(dy, "dy"), stream_of(dy)),
          "flb_gate_bwd");
  return {dx, dz};
}

struct GateFn : torch::autograd::Function<GateFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& z, bool keep8) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto out = gate_forward(x, z, keep8);
    if (keep8) ctx->save_for_backward({out[1], out[2], out[3], out[4]});
    else ctx->save_for_backward({x, z});
    return out[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    torch::autograd::variable_list out(3);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1]) = gate_backward(ctx->get_saved_variables(), g[0]);
    }
    return differentiable_once(std::move(out));
  }
};

Tensor sigmoid_gate(const Tensor& x, const Tensor& z, bool keep8) {
  for (const Opt& t : {Opt(x), Opt(z)}) no_tangent(t, "sigmoid_gate");
  if (c10::GradMode::is_enabled() && (x.requires_grad() || z.requires_grad())) return GateFn::apply(x, z, keep8);
  return gate_forward(x, z, false)[0];
}

// ---- 8-bit integer rows and their product -----------------------------------------------------------------

void no_gradient(const Opt& t, const char* what) {
  TORCH_CHECK(!(c10::GradMode::is_enabled() && wants_grad(t)), what, " has no gradient: call it under torch.no_grad()");
  no_tangent(t, what);
}

// codes [.., D] over rows that start every 16 bytes, and a scale each
std::pair<Tensor, Tensor> int8_buffers(const Tensor& x) {
  const int64_t D = x.size(-1), pitch = flb_code_pitch(D);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = pitch;
  Tensor codes = at::empty(shape, x.options().dtype(at::kChar));
  Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  return {pitch == D ? codes : codes.narrow(-1, 0, D), scale};
}

std::pair<Tensor, Tensor> quantize_int8(const Tensor& x_) {
  no_gradient(x_, "quantize_int8");
  const int dt = dtype_of(x_, "x");
  need_cuda(x_);
  TORCH_CHECK_VALUE(last_axis(x_, "x") >= 1, "x must have a last axis of at least one element");
  const c10::cuda::CUDAGuard guard(x_.device());
  auto [x, ldx] = rows_of(x_);
  auto [codes, scale] = int8_buffers(x);
  check(flb_int8_rows(x.data_ptr(), ldx, (int8_t*)codes.data_ptr(), (float*)scale.data_ptr(), rows_in(x), x.size(-1), dt, stream_of(x)),
        "flb_int8_rows");
  return {codes, scale};
}

std::pair<Tensor, Tensor> layer_norm_int8(const Tensor& x_, const Opt& weight, const Opt& bias, double eps) {
  for (const Opt& t : {Opt(x_), weight, bias}) no_gradient(t, "layer_norm_int8");
  const NormSizes n = check_norm(x_, weight, bias);
  const c10::cuda::CUDAGuard guard(x_.device());
  auto [x, ldx] = rows_of(x_);
  const Opt w = contiguous(weight), b = contiguous(bias);
  auto [codes, scale] = int8_buffers(x);
  check(flb_layer_norm_int8(x.data_ptr(), ldx, ptr(w), ptr(b), n.wdt, (int8_t*)codes.data_ptr(), (float*)scale.data_ptr(), n.G, n.R,
                            n.D, n.dt, (float)eps, stream_of(x)),
        "flb_layer_norm_int8");
  return {codes, scale};
}

// Codes as the product takes them: rows a multiple of 16 bytes apart, the first on 16 bytes; copied so if need be.
std::tuple<Tensor, int64_t> code_rows(const Tensor& codes, const Tensor& scale, const char* name) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat, name,
                   " must be int8 codes and float32 scales, not ", codes.scalar_type(), " and ", scale.scalar_type());
  TORCH_CHECK_VALUE(codes.dim() >= 1 && scale.sizes() == codes.sizes().slice(0, codes.dim() - 1), name, ": codes of shape ",
                    codes.sizes(), " with scales of shape ", scale.sizes());
  const int64_t K = codes.size(-1);
  if (codes.numel() == 0) return {codes, flb_code_pitch(K)};
  auto [t, pitch] = rows_of(codes);
  const int64_t rows = rows_in(t);
  if (rows == 1) pitch = flb_code_pitch(K);  // one row has no pitch of its own
  if (pitch % 16 == 0 && pitch >= K && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return {t, pitch};
  Tensor padded = at::empty({rows, flb_code_pitch(K)}, t.options());
  padded.narrow(1, 0, K).copy_(t.reshape({rows, K}));
  return {padded, flb_code_pitch(K)};
}

// x, or x_codes and x_scale with the output's type
Tensor int8_linear(const Opt& x_, const Opt& x_codes, const Opt& x_scale, const Tensor& w_codes, const Tensor& w_scale,
                   const Opt& bias_, std::optional<at::ScalarType> type, bool check_timeout) {
  for (const Opt& t : {x_, x_scale, Opt(w_scale), bias_}) no_gradient(t, "int8_linear");
  const Tensor& in = given(x_) ? *x_ : *x_codes;
  const at::ScalarType dtype = given(x_) ? in.scalar_type() : type.value_or(at::kBFloat16);
  const int dt = dtype_of(dtype, "x");
  need_cuda(in);
  for (const Opt& t : {Opt(w_codes), Opt(w_scale), x_scale, bias_}) same_device(in, t);
  const int64_t K = last_axis(in, "x"), M = rows_in(in);
  TORCH_CHECK_VALUE(w_codes.dim() == 2 && w_codes.size(1) == K && K >= 1, "a weight of shape ", w_codes.sizes(), " for x of shape ",
                    in.sizes());
  const int64_t N = w_codes.size(0);
  int bdt = dt;
  if (given(bias_)) {
    bdt = dtype_of(*bias_, "bias");
    TORCH_CHECK_TYPE(bdt == FLB_F32 || bdt == dt, "bias must be float32 or ", dtype, ", not ", bias_->scalar_type());
    TORCH_CHECK_VALUE(bias_->dim() == 1 && bias_->size(0) == N, "a bias of shape ", bias_->sizes(), " for ", N, " outputs");
  }
  const c10::cuda::CUDAGuard guard(in.device());
  std::vector<int64_t> shape = in.sizes().vec();
  shape.back() = N;
  Tensor out = at::empty(shape, in.options().dtype(dtype));
  auto [wc, ldw] = code_rows(w_codes, w_scale, "the weight");
  const Tensor ws_ = w_scale.contiguous();
  Opt x, xc, xs;
  int64_t ldx = K, ldc = 0;
  if (given(x_)) {
    auto [t, ld] = rows_of(*x_);
    x = t, ldx = ld;
  } else {
    auto [t, ld] = code_rows(*x_codes, *x_scale, "x");
    xc = t, ldc = ld;
    xs = x_scale->contiguous();
  }
  if (M == 0 || N == 0) return out;
  const Opt b = contiguous(bias_);
  const size_t need = flb_int8_linear_workspace_bytes(M, N, K, given(x) ? 0 : 1);
  Tensor ws = buffer(need, in);
  check(flb_int8_linear(ptr(x), ldx, (const int8_t*)ptr(xc), ldc, (const float*)ptr(xs), (const int8_t*)wc.data_ptr(), ldw,
                        (const float*)ws_.data_ptr(), ptr(b), bdt, out.data_ptr(), M, N, K, dt, ws.data_ptr(), need, check_timeout ? 1 : 0, stream_of(in)),
        "flb_int8_linear");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  const auto off = py::call_guard<py::gil_scoped_release>();
  m.def("rows_of", &rows_of);
  m.def("layer_norm", &layer_norm, off);
  m.def("norm_forward", &norm_forward, off);
  m.def("norm_backward", &norm_backward, off);
  m.def("pack8", &pack8, off);
  m.def("unpack8", [](const Tensor& c, const Tensor& e, std::vector<int64_t> shape, py::object dtype) {
    const auto t = torch::python::detail::py_object_to_dtype(dtype);
    py::gil_scoped_release release;
    return unpack8(c, e, std::move(shape), t);
  });
  m.def("gate_forward", &gate_forward, off);
  m.def("gate_backward", &gate_backward, off);
  m.def("sigmoid_gate", &sigmoid_gate, off);
  m.def("quantize_int8", &quantize_int8, off);
  m.def("layer_norm_int8", &layer_norm_int8, off);
  m.def("int8_linear", [](const Opt& x, const Opt& xc, const Opt& xs, const Tensor& wc, const Tensor& ws, const Opt& bias, py::object dtype,
                          bool check_timeout) {
    std::optional<at::ScalarType> t;
    if (!dtype.is_none()) t = torch::python::detail::py_object_to_dtype(dtype);
    py::gil_scoped_release release;
    return int8_linear(x, xc, xs, wc, ws, bias, t, check_timeout);
  });
}
