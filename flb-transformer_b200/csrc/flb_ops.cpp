// flb_ops: the row operators' torch side in C++: argument checks, buffers, streams, devices and autograd
// functions around the C ABI of libflb_b200.so. In C++ because a training step through a small row operator
// is bound by the host: as Python functions, forward and backward of a norm over 192 rows took 146 us on a B200
// machine, nearly all of it the interpreter's. The Python packages keep the operators' names, their
// documentation and their torch.func rules. There is no CPU path.
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
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

// ---- 8-bit floating-point rows and their product ----------------------------------------------------------------

// Codes of a matrix of `rows` rows of K, each row from 16 bytes on, and their powers of two
struct Fp8 {
  Tensor codes, exps;  // [rows, pitch], [groups of 128 rows, quads of blocks, 32, 4, 4]
};
Fp8 fp8_buffers(int64_t rows, int64_t K, const Tensor& like) {
  return {at::empty({rows, flb_code_pitch(K)}, like.options().dtype(at::kFloat8_e4m3fn)),
          at::empty({(rows + 127) / 128, (K + 511) / 512, 32, 4, 4}, like.options().dtype(at::kByte))};
}

// x's rows
Fp8 fp8_rows(const Tensor& x_) {
  const int dt = dtype_of(x_, "x");
  auto [x, ldx] = rows_of(x_);
  const int64_t K = x.size(-1), R = rows_in(x);
  Fp8 q = fp8_buffers(R, K, x);
  check(flb_fp8_rows(x.data_ptr(), ldx, q.codes.data_ptr(), (uint8_t*)q.exps.data_ptr(), R, K, dt, stream_of(x)), "flb_fp8_rows");
  return q;
}
// The product of x [M, K], or its codes, and a weight's [N, K] codes into out
void fp8_product(const Opt& x_, int64_t ldx, const Fp8& xq, int64_t ldc, const Fp8& w, int64_t ldw, const Opt& bias, const Tensor& out, int64_t M, int64_t N,
                 int64_t K, bool check_timeout) {
  if (M == 0 || N == 0) return;
  const bool from_x = given(x_);
  const size_t need = flb_fp8_linear_workspace_bytes(M, N, K, from_x ? 0 : 1);
  Tensor ws = buffer(need, out);
  check(flb_fp8_linear(ptr(x_), ldx, from_x ? nullptr : xq.codes.data_ptr(), ldc, from_x ? nullptr : (const uint8_t*)xq.exps.data_ptr(), w.codes.data_ptr(),
                       ldw, (const uint8_t*)w.exps.data_ptr(), ptr(bias), given(bias) ? dtype_of(*bias, "bias") : FLB_F32, out.data_ptr(), M, N, K,
                       dtype_of(out, "out"), ws.data_ptr(), need, check_timeout ? 1 : 0, stream_of(out)),
        "flb_fp8_linear");
}

std::pair<Tensor, Tensor> quantize_fp8(const Tensor& x) {
  no_gradient(x, "quantize_fp8");
  dtype_of(x, "x");
  need_cuda(x);
  TORCH_CHECK_VALUE(last_axis(x, "x") >= 1, "x must have a last axis of at least one element");
  const c10::cuda::CUDAGuard guard(x.device());
  Fp8 q = fp8_rows(x);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = q.codes.size(1);
  return {q.codes.view(shape).narrow(-1, 0, x.size(-1)), q.exps};
}

// Codes as the product takes them: rows a multiple of 16 bytes apart, the first on 16 bytes; copied so if need be.
std::tuple<Fp8, int64_t> fp8_operand(const Tensor& codes, const Tensor& exps, const char* name) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kFloat8_e4m3fn && exps.scalar_type() == at::kByte, name,
                   " must be float8_e4m3fn codes and uint8 powers of two, not ", codes.scalar_type(), " and ", exps.scalar_type());
  TORCH_CHECK_VALUE(codes.dim() >= 1 && codes.size(-1) >= 1, name, ": codes must have a last axis of at least one element");
  const int64_t K = codes.size(-1), R = rows_in(codes);
  TORCH_CHECK_VALUE(exps.numel() == (int64_t)flb_fp8_exps_bytes(R, K) && exps.is_contiguous() && (exps.numel() == 0 || reinterpret_cast<uintptr_t>(exps.data_ptr()) % 16 == 0),
                    name, ": powers of two of shape ", exps.sizes(), " are not those of codes of shape ", codes.sizes());
  if (codes.numel() == 0) return {Fp8{codes, exps}, flb_code_pitch(K)};
  auto [t, pitch] = rows_of(codes);
  if (R == 1) pitch = flb_code_pitch(K);  // one row has no pitch of its own
  if (pitch % 16 == 0 && pitch >= K && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return {Fp8{t, exps}, pitch};
  Tensor padded = at::empty({R, flb_code_pitch(K)}, t.options());
  padded.view(at::kByte).narrow(1, 0, K).copy_(t.reshape({R, K}).view(at::kByte));
  return {Fp8{padded, exps}, flb_code_pitch(K)};
}

void check_fp8(const Tensor& in, int64_t N, int64_t K, at::IntArrayRef weight, const Opt& bias) {
  TORCH_CHECK_VALUE(weight.size() == 2 && weight[1] == K && K >= 1, "a weight of shape ", weight, " for x of shape ", in.sizes());
  if (!given(bias)) return;
  same_device(in, bias);
  dtype_of(*bias, "bias");
  TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, "a bias of shape ", bias->sizes(), " for ", N, " outputs");
}

// x, or its codes with the output's type; a weight that is kept as codes
Tensor fp8_linear_kept(const Opt& x_, const Opt& x_codes, const Opt& x_exps, const Tensor& w_codes, const Tensor& w_exps, const Opt& bias_,
                       std::optional<at::ScalarType> type, bool check_timeout) {
  for (const Opt& t : {x_, bias_}) no_gradient(t, "fp8_linear with a weight kept in 8 bits");
  const Tensor& in = given(x_) ? *x_ : *x_codes;
  const at::ScalarType dtype = given(x_) ? in.scalar_type() : type.value_or(at::kBFloat16);
  dtype_of(dtype, "x");
  need_cuda(in);
  for (const Opt& t : {Opt(w_codes), Opt(w_exps), x_exps}) same_device(in, t);
  const int64_t K = last_axis(in, "x"), M = rows_in(in);
  check_fp8(in, w_codes.dim() == 2 ? w_codes.size(0) : 0, K, w_codes.sizes(), bias_);
  const int64_t N = w_codes.size(0);
  const c10::cuda::CUDAGuard guard(in.device());
  std::vector<int64_t> shape = in.sizes().vec();
  shape.back() = N;
  Tensor out = at::empty(shape, in.options().dtype(dtype));
  auto [w, ldw] = fp8_operand(w_codes, w_exps, "the weight");
  const Opt bias = contiguous(bias_);
  if (given(x_)) {
    auto [x, ldx] = rows_of(*x_);
    fp8_product(x, ldx, {}, 0, w, ldw, bias, out, M, N, K, check_timeout);
  } else {
    auto [xq, ldc] = fp8_operand(*x_codes, *x_exps, "x");
    fp8_product({}, 0, xq, ldc, w, ldw, bias, out, M, N, K, check_timeout);
  }
  return out;
}

// Several arrays in one buffer: a small training step is bound by the host, and an allocation costs it a microsecond.
struct Arena {
  size_t bytes = 0;
  size_t add(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) & ~(size_t)255;
    return at;
  }
};
struct Fp8Place {
  size_t codes, exps;
  Fp8Place(Arena& a, int64_t rows, int64_t K) : codes(a.add((size_t)rows * flb_code_pitch(K))), exps(a.add(flb_fp8_exps_bytes(rows, K))) {}
};
struct Fp8At {
  void* codes;
  uint8_t* exps;
  Fp8At(void* base, const Fp8Place& p) : codes((uint8_t*)base + p.codes), exps((uint8_t*)base + p.exps) {}
};
void fp8_codes(const Tensor& x_, const Fp8At& q) {
  auto [x, ldx] = rows_of(x_);
  check(flb_fp8_rows(x.data_ptr(), ldx, q.codes, q.exps, rows_in(x), x.size(-1), dtype_of(x, "x"), stream_of(x)), "flb_fp8_rows");
}
// along both axes, and with bias_grad the columns' sums
void fp8_codes2(const Tensor& x_, const Fp8At& q, const Fp8At& t, const Opt& bias_grad, void* ws, size_t need) {
  auto [x, ldx] = rows_of(x_);
  const int dt = dtype_of(x, "x");
  check(flb_fp8_rows2(x.data_ptr(), ldx, q.codes, q.exps, t.codes, t.exps, ptr(bias_grad), given(bias_grad) ? dtype_of(*bias_grad, "bias") : dt, rows_in(x),
                      x.size(-1), dt, ws, need, stream_of(x)),
        "flb_fp8_rows2");
}
void fp8_codes_product(const Fp8At& x, const Fp8At& w, const Opt& bias, const Tensor& out, int64_t M, int64_t N, int64_t K, void* ws, size_t need) {
  check(flb_fp8_linear(nullptr, 0, x.codes, flb_code_pitch(K), x.exps, w.codes, flb_code_pitch(K), w.exps, ptr(bias),
                       given(bias) ? dtype_of(*bias, "bias") : FLB_F32, out.data_ptr(), M, N, K, dtype_of(out, "out"), ws, need, 0, stream_of(out)),
        "flb_fp8_linear");
}

// A training step's products. x [M, K] and the weight [N, K] are kept for the backward pass as the 8-bit columns that it sums over.
struct Fp8LinearFn : torch::autograd::Function<Fp8LinearFn> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Opt& bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t K = x.size(-1), M = rows_in(x), N = weight.size(0);
    const bool for_dx = x.requires_grad(), for_dw = weight.requires_grad();
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = N;
    Tensor out = at::empty(shape, x.options()), columns;
    if (M && N) {
      Arena here, kept;
      const Fp8Place xq(here, M, K), wq(here, N, K);
      const size_t need = flb_fp8_linear_workspace_bytes(M, N, K, 1), ws = here.add(need);
      const Fp8Place xt(kept, for_dw ? K : 0, M), wt(kept, for_dx ? K : 0, N);
      const Tensor t = buffer(here.bytes, x);
      columns = buffer(kept.bytes, x);
      uint8_t* const at = (uint8_t*)t.data_ptr();
      void* const keep = columns.data_ptr();
      if (for_dw) fp8_codes2(x, {at, xq}, {keep, xt}, {}, nullptr, 0);
      else fp8_codes(x, {at, xq});
      if (for_dx) fp8_codes2(weight, {at, wq}, {keep, wt}, {}, nullptr, 0);
      else fp8_codes(weight, {at, wq});
      fp8_codes_product({at, xq}, {at, wq}, contiguous(bias), out, M, N, K, at + ws, need);
    }
    ctx->save_for_backward({columns});
    ctx->saved_data["sizes"] = std::vector<int64_t>{M, N, K, for_dx, for_dw, (int64_t)weight.scalar_type(), given(bias) ? (int64_t)bias->scalar_type() : -1};
    ctx->saved_data["x"] = x.sizes().vec();
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    torch::autograd::variable_list out(3);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const auto s = ctx->get_saved_variables();
      const auto sizes = ctx->saved_data["sizes"].toIntVector();
      const int64_t M = sizes[0], N = sizes[1], K = sizes[2];
      const bool for_dx = ctx->needs_input_grad(0), for_dw = ctx->needs_input_grad(1), for_db = sizes[6] >= 0 && ctx->needs_input_grad(2);
      const Tensor& dy = g[0];
      const c10::cuda::CUDAGuard guard(dy.device());
      const bool some = M && N;
      auto grad = [&](at::IntArrayRef shape, int64_t type) {
        const auto options = dy.options().dtype((at::ScalarType)type);
        return some ? at::empty(shape, options) : at::zeros(shape, options);
      };
      if (for_dx) out[0] = grad(ctx->saved_data["x"].toIntVector(), (int64_t)dy.scalar_type());
      if (for_dw) out[1] = grad({N, K}, sizes[5]);
      if (for_db) out[2] = grad({N}, sizes[6]);
      if (some) {
        // (one workspace for both products: the second starts when the first has ended)
        Arena here, kept;
        const Fp8Place xt(kept, sizes[4] ? K : 0, M), wt(kept, sizes[3] ? K : 0, N);
        const bool both = for_dw || for_db;
        const Fp8Place q(here, M, N), t(here, both ? N : 0, M);
        const size_t sums_need = for_db ? flb_fp8_rows2_workspace_bytes(M, N) : 0, sums = here.add(sums_need);
        const size_t dx_need = for_dx ? flb_fp8_linear_workspace_bytes(M, K, N, 1) : 0, dw_need = for_dw ? flb_fp8_linear_workspace_bytes(N, K, M, 1) : 0;
        const size_t need = std::max(dx_need, dw_need), ws = here.add(need);
        const Tensor held = buffer(here.bytes, dy);
        uint8_t* const at = (uint8_t*)held.data_ptr();
        void* const keep = s[0].data_ptr();
        if (both) fp8_codes2(dy, {at, q}, {at, t}, for_db ? Opt(out[2]) : Opt(), at + sums, sums_need);
        else fp8_codes(dy, {at, q});
        if (for_dx) fp8_codes_product({at, q}, {keep, wt}, {}, out[0], M, K, N, at + ws, need);
        if (for_dw) fp8_codes_product({at, t}, {keep, xt}, {}, out[1], N, K, M, at + ws, need);
      }
    }
    return differentiable_once(std::move(out));
  }
};

Tensor fp8_linear(const Tensor& x, const Tensor& weight, const Opt& bias) {
  for (const Opt& t : {Opt(x), Opt(weight), bias}) no_tangent(t, "fp8_linear");
  dtype_of(x, "x");
  dtype_of(weight, "weight");
  need_cuda(x);
  same_device(x, weight);
  check_fp8(x, weight.dim() == 2 ? weight.size(0) : 0, last_axis(x, "x"), weight.sizes(), bias);
  if (c10::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(bias))) return Fp8LinearFn::apply(x, weight, bias);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t K = x.size(-1), M = rows_in(x), N = weight.size(0);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  Tensor out = at::empty(shape, x.options());
  if (M == 0 || N == 0) return out;
  auto [rows, ldx] = rows_of(x);
  const Fp8 wq = fp8_rows(weight);
  fp8_product(rows, ldx, {}, 0, wq, flb_code_pitch(K), contiguous(bias), out, M, N, K, false);
  return out;
}

// ---- a token from logits ------------------------------------------------------------------------------------

// A setting for each row, or none.
Opt row_setting(const Opt& t, const Tensor& logits, at::ScalarType type, const char* name) {
  if (!given(t)) return Opt();
  same_device(logits, t);
  TORCH_CHECK_TYPE(t->scalar_type() == type, name, " must be a number or a tensor of ", type, ", not of ", t->scalar_type());
  TORCH_CHECK_VALUE(t->sizes() == logits.sizes().slice(0, logits.dim() - 1), name, " of shape ", t->sizes(), " for logits of shape ",
                    logits.sizes());
  return t->contiguous();
}

Tensor sample(const Tensor& logits_, const Tensor& u_, const Opt& temperature_, double temperature_all, const Opt& top_k_, int64_t top_k_all,
              const Opt& top_p_, double top_p_all, const Opt& min_p_, double min_p_all) {
  const int dt = dtype_of(logits_, "logits");
  need_cuda(logits_);
  TORCH_CHECK_VALUE(last_axis(logits_, "logits") >= 1, "logits must have a last axis of at least one element");
  const bool u64 = u_.scalar_type() == at::kDouble;
  const c10::cuda::CUDAGuard guard(logits_.device());
  const Opt u = row_setting(u_, logits_, u64 ? at::kDouble : at::kFloat, "u");
  const Opt temperature = row_setting(temperature_, logits_, at::kFloat, "temperature"), top_k = row_setting(top_k_, logits_, at::kLong, "top_k");
  const Opt top_p = row_setting(top_p_, logits_, at::kFloat, "top_p"), min_p = row_setting(min_p_, logits_, at::kFloat, "min_p");
  auto [x, ld] = rows_of(logits_);
  Tensor token = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kLong));
  check(flb_sample(x.data_ptr(), ld, ptr(u), u64, token.data_ptr<int64_t>(), rows_in(x), x.size(-1), dt, (const float*)ptr(temperature),
                   temperature_all, (const int64_t*)ptr(top_k), top_k_all, (const float*)ptr(top_p), top_p_all, (const float*)ptr(min_p),
                   min_p_all, stream_of(x)),
        "flb_sample");
  return token;
}

// ---- AdamW ----------------------------------------------------------------------------------------------------

// Elements in memory's order, one after the other: what a kernel that goes by addresses needs.
void need_dense(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense(), "AdamW: ", name, " of shape ", t.sizes(), " and strides ", t.strides(),
                    " has gaps or shares elements");
}
void need_codes(const Tensor& codes, const Tensor& exps, const Tensor& p) {
  const int64_t blocks = (p.numel() + 127) / 128;
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && exps.scalar_type() == at::kByte && codes.numel() == blocks * 128 &&
                        exps.numel() == blocks && codes.is_contiguous() && exps.is_contiguous(),
                    "AdamW: a moment's codes and exponents are not those of a parameter of shape ", p.sizes());
  same_device(p, codes);
  same_device(p, exps);
}
bool same_layout(const Tensor& a, const Tensor& b) { return a.sizes() == b.sizes() && (a.numel() <= 1 || a.strides() == b.strides()); }

// The optimizer's state goes by Python objects: read here, since a loop over parameters in Python took twice the time of all checks and the launch
// (135 us a step of 48 parameters, 50 so).
const Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(o && THPVariable_Check(o), "AdamW: a parameter's state has no tensor \"", name, "\"");
  return THPVariable_Unpack(o);
}
struct Names {
  PyObject *step, *m, *v, *m_exps, *v_exps, *strides;
};
const Names& names() {
  static const Names n{PyUnicode_InternFromString("step"), PyUnicode_InternFromString("exp_avg"), PyUnicode_InternFromString("exp_avg_sq"),
                       PyUnicode_InternFromString("exp_avg_exps"), PyUnicode_InternFromString("exp_avg_sq_exps"),
                       PyUnicode_InternFromString("strides")};
  return n;
}
// state[p], borrowed; null where there is none or it is empty
PyObject* state_of(PyObject* state, PyObject* p) {
  PyObject* const s = PyDict_GetItemWithError(state, p);
  if (!s && PyErr_Occurred()) throw pybind11::error_already_set();
  return s && PyDict_Check(s) && PyDict_Size(s) > 0 ? s : nullptr;
}
const Tensor& get(PyObject* s, PyObject* name, const char* text) { return tensor_of(PyDict_GetItemWithError(s, name), text); }

// Codes lie as their parameter did when they were made: the state of one that is not contiguous has its strides.
void need_order(PyObject* s, const Tensor& p) {
  PyObject* const strides = PyDict_GetItemWithError(s, names().strides);
  if (!strides && PyErr_Occurred()) throw pybind11::error_already_set();
  bool same = strides ? PyTuple_Check(strides) && PyTuple_GET_SIZE(strides) == p.dim() : p.is_contiguous();
  for (int64_t i = 0; strides && same && i < p.dim(); ++i) {
    const int64_t stride = PyLong_AsLongLong(PyTuple_GET_ITEM(strides, i));
    if (stride == -1 && PyErr_Occurred()) throw pybind11::error_already_set();
    same = p.size(i) == 1 || stride == p.stride(i);
  }
  TORCH_CHECK_VALUE(same, "AdamW: 8-bit moments are not laid out as their parameter, of shape ", p.sizes(), " and strides ", p.strides());
}

// The tensors of one device and type, one kernel's.
struct Together {
  at::Device device;
  at::ScalarType type;
  std::vector<flb_adamw_tensor> t;
  std::vector<Tensor> held;  // gradients in their parameters' order, until the launch
  Tensor like;
};

// A step of every parameter that has a gradient. Returns those that have no state yet: then nothing has been done.
pybind11::list adamw(pybind11::list params, pybind11::dict state, int64_t bits, double lr, const Opt& lr_device, double b1, double b2, double eps,
                     double decay, uint32_t seed, pybind11::dict counters) {
  // (a group's lr may have been put in another's place since the optimizer was made)
  TORCH_CHECK_VALUE(!given(lr_device) || (lr_device->scalar_type() == at::kFloat && lr_device->numel() == 1),
                    "AdamW: lr on the device must be one float32, not ", given(lr_device) ? lr_device->numel() : 0, " of ",
                    given(lr_device) ? lr_device->scalar_type() : at::kFloat);
  pybind11::list missing;
  std::vector<Together> all;
  std::vector<Tensor> written;
  for (pybind11::handle h : params) {
    const Tensor& p = tensor_of(h.ptr(), "parameter");
    Tensor g = p.grad();
    if (!g.defined()) continue;
    PyObject* const s = state_of(state.ptr(), h.ptr());
    if (!s) {
      missing.append(h);
      continue;
    }
    if (pybind11::len(missing)) continue;
    need_cuda(p);
    dtype_of(p, "a parameter");
    need_dense(p, "a parameter");
    Together* to = nullptr;
    for (Together& x : all)
      if (x.device == p.device() && x.type == p.scalar_type()) to = &x;
    if (!to) {
      all.push_back({p.device(), p.scalar_type(), {}, {}, p});
      to = &all.back();
    }
    same_device(p, g);
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, "AdamW: sparse gradients are not supported");
    TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "AdamW: a gradient of ", g.scalar_type(), " for a parameter of ", p.scalar_type());
    TORCH_CHECK_VALUE(g.sizes() == p.sizes(), "AdamW: a gradient of shape ", g.sizes(), " for a parameter of shape ", p.sizes());
    if (!same_layout(g, p)) {
      const c10::cuda::CUDAGuard guard(p.device());
      g = at::empty_like(p).copy_(g);
      to->held.push_back(g);
    }
    const Names& n = names();
    const Tensor &step = get(s, n.step, "step"), &m = get(s, n.m, "exp_avg"), &v = get(s, n.v, "exp_avg_sq");
    flb_adamw_tensor t{p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), nullptr, nullptr, nullptr, p.numel()};
    if (bits == 8) {
      const Tensor &me = get(s, n.m_exps, "exp_avg_exps"), &ve = get(s, n.v_exps, "exp_avg_sq_exps");
      need_codes(m, me, p);
      need_codes(v, ve, p);
      need_order(s, p);
      t.m_exps = (uint8_t*)me.data_ptr(), t.v_exps = (uint8_t*)ve.data_ptr();
      written.push_back(me), written.push_back(ve);
    } else {
      for (const Tensor* x : {&m, &v}) {
        same_device(p, *x);
        TORCH_CHECK_VALUE(x->scalar_type() == at::kFloat && same_layout(*x, p), "AdamW: a moment is not a float32 tensor laid out as its parameter");
      }
    }
    same_device(p, step);
    TORCH_CHECK_VALUE(step.scalar_type() == at::kLong && step.numel() == 1, "AdamW: step must be one int64");
    t.step = step.data_ptr<int64_t>();
    to->t.push_back(t);
    for (const Tensor* x : {&p, &m, &v, &step}) written.push_back(*x);
  }
  if (pybind11::len(missing)) return missing;
  std::vector<Tensor> words;
  for (Together& x : all) {
    same_device(x.like, lr_device);
    const c10::cuda::CUDAGuard guard(x.device);
    // A word of the kernel's own on each device, zero between steps. Not made in a capture, which would only record that it is cleared.
    const pybind11::int_ key(x.device.index());
    if (!counters.contains(key)) {
      TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None,
                  "AdamW: the first step on a device makes a word of the kernel's there: take one before the capture");
      counters[key] = pybind11::cast(at::zeros({1}, x.like.options().dtype(at::kInt).requires_grad(false)));
    }
    words.push_back(counters[key].cast<Tensor>());
  }
  for (size_t i = 0; i < all.size(); ++i) {
    Together& x = all[i];
    const c10::cuda::CUDAGuard guard(x.device);
    check(flb_adamw(x.t.data(), (int64_t)x.t.size(), dtype_of(x.type, "a parameter"), (int)bits, lr, (const float*)ptr(lr_device), b1, b2, eps, decay, seed,
                    (uint32_t*)words[i].data_ptr(), stream_of(x.like)),
          "flb_adamw");
  }
  // written behind autograd's back: a graph that still needs the old values is told
  for (const Tensor& x : written) x.unsafeGetTensorImpl()->bump_version();
  return missing;
}

// The moments of parameters that have 8-bit state, as pairs: into those of `out` from its place `at` on, or new ones.
pybind11::list adamw_moments(pybind11::list params, pybind11::dict state, pybind11::object out, size_t at) {
  pybind11::list found;
  std::vector<Together> all;
  std::vector<Tensor> written;
  for (pybind11::handle h : params) {
    PyObject* const s = state_of(state.ptr(), h.ptr());
    if (!s) continue;
    const Tensor& p = tensor_of(h.ptr(), "parameter");
    need_cuda(p);
    const c10::cuda::CUDAGuard guard(p.device());
    Tensor pair[2];
    if (out.is_none()) {
      for (Tensor& x : pair) x = at::empty_like(p, p.options().dtype(at::kFloat).requires_grad(false));
    } else {
      const pybind11::object given = out[pybind11::int_(at++)];
      for (int i = 0; i < 2; ++i) {
        pair[i] = pybind11::object(given[pybind11::int_(i)]).cast<Tensor>();
        same_device(p, pair[i]);
        TORCH_CHECK_VALUE(pair[i].scalar_type() == at::kFloat && same_layout(pair[i], p), "AdamW: moments go to float32 tensors laid out as their parameters");
      }
    }
    const Names& n = names();
    const Tensor &m = get(s, n.m, "exp_avg"), &v = get(s, n.v, "exp_avg_sq"), &me = get(s, n.m_exps, "exp_avg_exps"), &ve = get(s, n.v_exps, "exp_avg_sq_exps");
    need_codes(m, me, p);
    need_codes(v, ve, p);
    need_order(s, p);
    Together* to = nullptr;
    for (Together& x : all)
      if (x.device == p.device()) to = &x;
    if (!to) {
      all.push_back({p.device(), at::kFloat, {}, {}, p});
      to = &all.back();
    }
    to->t.push_back(flb_adamw_tensor{pair[0].data_ptr(), pair[1].data_ptr(), m.data_ptr(), v.data_ptr(), (uint8_t*)me.data_ptr(), (uint8_t*)ve.data_ptr(),
                                     nullptr, p.numel()});
    for (const Tensor& x : pair) written.push_back(x);
    found.append(pybind11::make_tuple(pair[0], pair[1]));
  }
  for (Together& x : all) {
    const c10::cuda::CUDAGuard guard(x.device);
    check(flb_adamw_moments(x.t.data(), (int64_t)x.t.size(), stream_of(x.like)), "flb_adamw_moments");
  }
  for (const Tensor& x : written) x.unsafeGetTensorImpl()->bump_version();
  return found;
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
  m.def("quantize_fp8", &quantize_fp8, off);
  m.def("fp8_linear", &fp8_linear, off);
  m.def("fp8_linear_kept", [](const Opt& x, const Opt& xc, const Opt& xe, const Tensor& wc, const Tensor& we, const Opt& bias, py::object dtype,
                              bool check_timeout) {
    std::optional<at::ScalarType> t;
    if (!dtype.is_none()) t = torch::python::detail::py_object_to_dtype(dtype);
    py::gil_scoped_release release;
    return fp8_linear_kept(x, xc, xe, wc, we, bias, t, check_timeout);
  });
  m.def("sample", &sample, off);
  m.def("adamw", &adamw);
  m.def("adamw_moments", &adamw_moments);
  m.def("int8_linear", [](const Opt& x, const Opt& xc, const Opt& xs, const Tensor& wc, const Tensor& ws, const Opt& bias, py::object dtype,
                          bool check_timeout) {
    std::optional<at::ScalarType> t;
    if (!dtype.is_none()) t = torch::python::detail::py_object_to_dtype(dtype);
    py::gil_scoped_release release;
    return int8_linear(x, xc, xs, wc, ws, bias, t, check_timeout);
  });
}
