// extern "C" boundary of the operators around a model's head: the choice of a token from its logits, and AdamW.
#include <cmath>
#include "common.cuh"

namespace flb {

int sample(const void* logits, int64_t ld, const void* u, bool u64, int64_t* token, int64_t rows, int64_t V, int dtype, const float* temperature,
           const int64_t* top_k, const float* top_p, const float* min_p, double temperature1, int64_t top_k1, double top_p1, double min_p1,
           cudaStream_t s);
int adamw(const flb_adamw_tensor* t, int64_t count, int dtype, int state_bits, double lr, const float* lr_device, double b1, double b2,
          double eps, double decay, uint32_t seed, uint32_t* counter, cudaStream_t s);
int adamw_moments(const flb_adamw_tensor* t, int64_t count, cudaStream_t s);

namespace {

bool off(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; }

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

}  // namespace
}  // namespace flb

using namespace flb;

extern "C" {

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
