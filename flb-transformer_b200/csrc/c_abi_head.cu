// extern "C" boundary of the operators around a model's head: products in 8-bit floating point, the choice of a token from
// logits, and AdamW.
#include <cmath>
#include "fp8.cuh"

namespace flb {

int fp8_rows(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int64_t R, int64_t K, int dtype, bool whole, uint32_t* zero, int n_zero,
             cudaStream_t s);
int fp8_rows2(const void* x, int64_t ldx, int8_t* codes, uint8_t* exps, int8_t* codes_t, uint8_t* exps_t, float* sums, void* bias_grad,
              int bias_dtype, int64_t R, int64_t C, int dtype, cudaStream_t s);
size_t fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise);
int fp8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const uint8_t* x_exps, const int8_t* w_codes, int64_t ldw,
               const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int dtype, void* ws,
               int check_timeout, int drop, uint32_t limit, cudaStream_t s);
int sample(const void* logits, int64_t ld, const void* u, bool u64, int64_t* token, int64_t rows, int64_t V, int dtype, const float* temperature,
           const int64_t* top_k, const float* top_p, const float* min_p, double temperature1, int64_t top_k1, double top_p1, double min_p1,
           cudaStream_t s);
int adamw(const flb_adamw_tensor* t, int64_t count, int dtype, int state_bits, double lr, const float* lr_device, double b1, double b2,
          double eps, double decay, uint32_t seed, uint32_t* counter, cudaStream_t s);
int adamw_moments(const flb_adamw_tensor* t, int64_t count, cudaStream_t s);

namespace {

bool off(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; }

// Sizes of rows of codes: within what grids, tensor maps and 32-bit coordinates hold.
int check_codes(const char* what, int64_t R, int64_t K) {
  const std::string at(what);
  if (R < 0 || K < 1) return fail(FLB_ERR_SHAPE, at + ": rows >= 0 of K >= 1 required");
  if (K > (1 << 30)) return fail(FLB_ERR_UNSUPPORTED, at + ": rows wider than 2^30 are not supported");
  if (R > INT32_MAX - 1024 || (R > 0 && K > ((int64_t)1 << 42) / R)) return fail(FLB_ERR_SHAPE, at + ": too many rows");
  return FLB_OK;
}

// What a step and reading the moments ask of each tensor. elem: bytes of an element of p and g.
int check_tensors(const char* what, const flb_adamw_tensor* t, int64_t count, size_t elem, bool codes, bool steps) {
  const std::string at(what);
  if (count < 0 || (count > 0 && !t)) return fail(FLB_ERR_SHAPE, at + ": bad tensor list");
  for (int64_t i = 0; i < count; ++i) {
    const flb_adamw_tensor& s = t[i];
    if (s.n < 0 || s.n > ((int64_t)1 << 40)) return fail(FLB_ERR_SHAPE, at + ": bad element count");
    if (steps && !s.step) return fail(FLB_ERR_SHAPE, at + ": null step");
    if (steps && off(s.step, 8)) return fail(FLB_ERR_ALIGN, at + ": step must be 8-byte aligned");
    if (s.n == 0) continue;
    if (!s.p || !s.g || !s.m || !s.v) return fail(FLB_ERR_SHAPE, at + ": null tensor");
    if (codes && (!s.m_exps || !s.v_exps)) return fail(FLB_ERR_SHAPE, at + ": codes need their exponents");
    if (off(s.p, elem) || off(s.g, elem) || off(s.m, 4) || off(s.v, 4))
      return fail(FLB_ERR_ALIGN, at + ": pointers must be aligned to their element size, codes to 4 bytes");
  }
  return FLB_OK;
}

int fp8_linear_checked(const void* x, int64_t ldx, const void* x_codes, int64_t ldc, const uint8_t* x_exps, const void* w_codes, int64_t ldw,
                       const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N, int64_t K, int dtype,
                       void* workspace, size_t workspace_bytes, int check_timeout, int drop, uint32_t limit, void* stream) {
  const size_t es = (size_t)dtype_size(dtype);
  if (es == 0 || (bias && dtype_size(bias_dtype) == 0)) return fail(FLB_ERR_DTYPE, "fp8_linear: dtype must be f32, f16 or bf16");
  int st = check_codes("fp8_linear", M, K);
  if (st == FLB_OK) st = check_codes("fp8_linear", N, K);
  if (st != FLB_OK) return st;
  if (M > 0 && N > ((int64_t)1 << 42) / M) return fail(FLB_ERR_SHAPE, "fp8_linear: too many outputs");
  if (M == 0 || N == 0) return FLB_OK;
  if (!x == !x_codes || !x_codes != !x_exps) return fail(FLB_ERR_SHAPE, "fp8_linear: either x, or x_codes and x_exps");
  if (!w_codes || !w_exps || !out) return fail(FLB_ERR_SHAPE, "fp8_linear: null weight or out");
  if (x ? ldx < 0 : ldc < K) return fail(FLB_ERR_SHAPE, "fp8_linear: bad row pitch of x");
  if (ldw < K) return fail(FLB_ERR_SHAPE, "fp8_linear: bad row pitch of the weight");
  if (off(w_codes, 16) || off(w_exps, 16) || ldw % 16 || (x_codes && (off(x_codes, 16) || off(x_exps, 16) || ldc % 16)))
    return fail(FLB_ERR_ALIGN, "fp8_linear: codes must start every row on 16 bytes, and exps lie on 16");
  if (off(x, es) || off(out, es) || off(bias, bias ? (size_t)dtype_size(bias_dtype) : 1))
    return fail(FLB_ERR_ALIGN, "fp8_linear: pointers must be aligned to their element size");
  if (!workspace || workspace_bytes < fp8_linear_workspace_bytes(M, N, K, x != nullptr))
    return fail(FLB_ERR_WORKSPACE, "fp8_linear: workspace smaller than flb_fp8_linear_workspace_bytes()");
  if (off(workspace, 256)) return fail(FLB_ERR_ALIGN, "fp8_linear: workspace must be 256-byte aligned");
  if (check_timeout) {
    cudaStreamCaptureStatus capture;
    if ((st = check_cuda(cudaStreamIsCapturing(as_stream(stream), &capture), "fp8_linear capture status")) != FLB_OK) return st;
    if (capture != cudaStreamCaptureStatusNone)
      return fail(FLB_ERR_UNSUPPORTED, "fp8_linear: check_timeout waits for the product, which a stream capture does not allow");
  }
  return fp8_linear(x, ldx, static_cast<const int8_t*>(x_codes), ldc, x_exps, static_cast<const int8_t*>(w_codes), ldw, w_exps, bias, bias_dtype, out, M,
                    N, K, dtype, workspace, check_timeout, drop, limit, as_stream(stream));
}

}  // namespace
}  // namespace flb

using namespace flb;

extern "C" {

size_t flb_fp8_exps_bytes(int64_t R, int64_t K) { return R < 1 || K < 1 ? 0 : (size_t)fp8::exps_bytes(R, K); }

int flb_fp8_rows(const void* x, int64_t ldx, void* codes, uint8_t* exps, int64_t R, int64_t K, int dtype, void* stream) {
  const size_t es = (size_t)dtype_size(dtype);
  if (es == 0) return fail(FLB_ERR_DTYPE, "fp8_rows: dtype must be f32, f16 or bf16");
  const int st = check_codes("fp8_rows", R, K);
  if (st != FLB_OK || R == 0) return st;
  if (!x || !codes || !exps || ldx < 0) return fail(FLB_ERR_SHAPE, "fp8_rows: null x, codes or exps, or a negative pitch");
  if (off(x, es) || off(codes, 16) || off(exps, 16)) return fail(FLB_ERR_ALIGN, "fp8_rows: codes and exps must be 16-byte aligned, x to its elements");
  return fp8_rows(x, ldx, static_cast<int8_t*>(codes), exps, R, K, dtype, true, nullptr, 0, as_stream(stream));
}

size_t flb_fp8_rows2_workspace_bytes(int64_t R, int64_t C) { return R < 1 || C < 1 ? 0 : (size_t)(fp8::blocks_of(R) * C) * 4; }

int flb_fp8_rows2(const void* x, int64_t ldx, void* codes, uint8_t* exps, void* codes_t, uint8_t* exps_t, void* bias_grad,
                  int bias_dtype, int64_t R, int64_t C, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const size_t es = (size_t)dtype_size(dtype);
  if (es == 0 || (bias_grad && dtype_size(bias_dtype) == 0)) return fail(FLB_ERR_DTYPE, "fp8_rows2: dtype must be f32, f16 or bf16");
  int st = check_codes("fp8_rows2", R, C);
  if (st == FLB_OK && R > 0) st = check_codes("fp8_rows2", C, R);
  if (st != FLB_OK || R == 0) return st;
  if (!x || !codes || !exps || !codes_t || !exps_t || ldx < 0) return fail(FLB_ERR_SHAPE, "fp8_rows2: null x, codes or exps, or a negative pitch");
  if (off(x, es) || off(codes, 16) || off(exps, 16) || off(codes_t, 16) || off(exps_t, 16) ||
      (bias_grad && off(bias_grad, (size_t)dtype_size(bias_dtype))))
    return fail(FLB_ERR_ALIGN, "fp8_rows2: codes and exps must be 16-byte aligned, x and bias_grad to their elements");
  if (bias_grad && (!workspace || workspace_bytes < flb_fp8_rows2_workspace_bytes(R, C)))
    return fail(FLB_ERR_WORKSPACE, "fp8_rows2: workspace smaller than flb_fp8_rows2_workspace_bytes()");
  if (bias_grad && off(workspace, 16)) return fail(FLB_ERR_ALIGN, "fp8_rows2: workspace must be 16-byte aligned");
  return fp8_rows2(x, ldx, static_cast<int8_t*>(codes), exps, static_cast<int8_t*>(codes_t), exps_t,
                   bias_grad ? static_cast<float*>(workspace) : nullptr, bias_grad, bias_dtype, R, C, dtype, as_stream(stream));
}

size_t flb_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_is_codes) {
  if (M < 1 || N < 1 || check_codes("fp8_linear", M, K) != FLB_OK || check_codes("fp8_linear", N, K) != FLB_OK || N > ((int64_t)1 << 42) / M) return 0;
  return fp8_linear_workspace_bytes(M, N, K, !x_is_codes);
}

int flb_fp8_linear(const void* x, int64_t ldx, const void* x_codes, int64_t ldc, const uint8_t* x_exps, const void* w_codes,
                   int64_t ldw, const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                   int64_t K, int dtype, void* workspace, size_t workspace_bytes, int check_timeout, void* stream) {
  return fp8_linear_checked(x, ldx, x_codes, ldc, x_exps, w_codes, ldw, w_exps, bias, bias_dtype, out, M, N, K, dtype, workspace, workspace_bytes,
                            check_timeout, -1, 0, stream);
}

int flb_fp8_linear_wait_test(const void* x, int64_t ldx, const void* x_codes, int64_t ldc, const uint8_t* x_exps, const void* w_codes,
                             int64_t ldw, const uint8_t* w_exps, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                             int64_t K, int dtype, void* workspace, size_t workspace_bytes, int check_timeout, int64_t drop_step,
                             uint32_t spin_limit, void* stream) {
  if (drop_step < -1 || drop_step > INT32_MAX || spin_limit == 0) return fail(FLB_ERR_SHAPE, "fp8_linear_wait_test: bad drop_step or spin_limit");
  return fp8_linear_checked(x, ldx, x_codes, ldc, x_exps, w_codes, ldw, w_exps, bias, bias_dtype, out, M, N, K, dtype, workspace, workspace_bytes,
                            check_timeout, (int)drop_step, spin_limit, stream);
}

int flb_sample(const void* logits, int64_t ld, const void* u, int u_is_f64, int64_t* token, int64_t rows, int64_t V, int dtype,
               const float* temperature, double temperature_all, const int64_t* top_k, int64_t top_k_all, const float* top_p,
               double top_p_all, const float* min_p, double min_p_all, void* stream) {
  const size_t es = (size_t)dtype_size(dtype);
  if (es == 0) return fail(FLB_ERR_DTYPE, "sample: dtype must be f32, f16 or bf16");
  if (rows < 0 || V < 1 || ld < 0) return fail(FLB_ERR_SHAPE, "sample: rows, ld >= 0 and V >= 1 required");
  if (V > 262144) return fail(FLB_ERR_UNSUPPORTED, "sample: vocabularies larger than 262144 are not supported");
  if (rows > (1 << 27)) return fail(FLB_ERR_SHAPE, "sample: too many rows");
  if (rows == 0) return FLB_OK;
  if (!logits || !u || !token) return fail(FLB_ERR_SHAPE, "sample: null logits, u or token");
  if (off(logits, es) || off(u, u_is_f64 ? 8 : 4) || off(token, 8) || off(temperature, 4) || off(top_k, 8) || off(top_p, 4) || off(min_p, 4))
    return fail(FLB_ERR_ALIGN, "sample: pointers must be aligned to their element size");
  return sample(logits, ld, u, u_is_f64 != 0, token, rows, V, dtype, temperature, top_k, top_p, min_p, temperature_all, top_k_all, top_p_all,
                min_p_all, as_stream(stream));
}

int flb_adamw(const flb_adamw_tensor* tensors, int64_t count, int dtype, int state_bits, double lr, const float* lr_device,
              double beta1, double beta2, double eps, double weight_decay, uint32_t seed, uint32_t* counter, void* stream) {
  const size_t es = (size_t)dtype_size(dtype);
  if (es == 0) return fail(FLB_ERR_DTYPE, "adamw: dtype must be f32, f16 or bf16");
  if (state_bits != 8 && state_bits != 32) return fail(FLB_ERR_UNSUPPORTED, "adamw: moments are held in 8 or 32 bits");
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1)) return fail(FLB_ERR_UNSUPPORTED, "adamw: betas must be at least 0 and below 1");
  const int st = check_tensors("adamw", tensors, count, es, state_bits == 8, true);
  if (st != FLB_OK || count == 0) return st;
  if (!counter) return fail(FLB_ERR_WORKSPACE, "adamw: null counter");
  if (off(counter, 4) || off(lr_device, 4)) return fail(FLB_ERR_ALIGN, "adamw: counter and lr must be 4-byte aligned");
  return adamw(tensors, count, dtype, state_bits, lr, lr_device, beta1, beta2, eps, weight_decay, seed, counter, as_stream(stream));
}

int flb_adamw_moments(const flb_adamw_tensor* tensors, int64_t count, void* stream) {
  const int st = check_tensors("adamw_moments", tensors, count, 4, true, false);
  return st != FLB_OK ? st : adamw_moments(tensors, count, as_stream(stream));
}

}  // extern "C"
