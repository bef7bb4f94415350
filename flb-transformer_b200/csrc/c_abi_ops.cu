// extern "C" boundary of the row operators (LayerNorm, the 8-bit kept form, the sigmoid gate) and of the 8-bit
// integer product.
#include "common.cuh"
#include "rows.cuh"

namespace flb {

int layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, void* y, float* mean,
                   float* rstd, int8_t* codes, uint8_t* exps, int64_t G, int64_t R, int64_t D, int dtype, float eps,
                   cudaStream_t s);
size_t layer_norm_bwd_workspace_bytes(int64_t G, int64_t R, int64_t D);
int layer_norm_bwd(const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps, const float* mean,
                   const float* rstd, const void* w, int wdtype, const void* dy, void* dx, void* dw, void* db, int64_t G,
                   int64_t R, int64_t D, int dtype, void* ws, cudaStream_t s);
int layer_norm_int8(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, int8_t* codes, float* scale,
                    int64_t G, int64_t R, int64_t D, int dtype, float eps, cudaStream_t s);
int int8_rows(const void* x, int64_t ldx, int8_t* codes, float* scale, int64_t R, int64_t D, int dtype, uint32_t* zero,
              int64_t n_zero, cudaStream_t s);
size_t int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, bool quantise);
int int8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale, const int8_t* w_codes,
                int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                int64_t K, int dtype, void* ws, int check_timeout, int drop, uint32_t limit, cudaStream_t s);
int pack8(const void* x, int8_t* codes, uint8_t* exps, int64_t R, int64_t D, int dtype, cudaStream_t s);
int unpack8(const int8_t* codes, const uint8_t* exps, void* out, int64_t R, int64_t D, int dtype, cudaStream_t s);
int gate_fwd(const void* x, const void* z, void* y, int8_t* cx, uint8_t* ex, int8_t* cz, uint8_t* ez, int64_t R,
             int64_t D, int dtype, cudaStream_t s);
int gate_bwd(const void* x, const void* z, const int8_t* cx, const uint8_t* ex, const int8_t* cz, const uint8_t* ez,
             const void* dy, void* dx, void* dz, int64_t R, int64_t D, int dtype, cudaStream_t s);

namespace {

bool off(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; }

// Sizes, dtypes and the parts of rows that every LayerNorm entry has. *empty: nothing to read or write.
int check_norm(const char* what, const void* w, const void* b, int wdtype, int64_t G, int64_t R, int64_t D,
               int64_t ldx, int dtype, int64_t widest, bool* empty) {
  const std::string at(what);
  if (dtype_size(dtype) == 0) return fail(FLB_ERR_DTYPE, at + ": dtype must be f32, f16 or bf16");
  if ((w || b) && wdtype != FLB_F32 && wdtype != dtype)
    return fail(FLB_ERR_DTYPE, at + ": weight and bias must be float32 or of the rows' dtype");
  if (G < 0 || R < 0 || D < 1 || ldx < 0) return fail(FLB_ERR_SHAPE, at + ": G, R, ldx >= 0 and D >= 1 required");
  if (D > widest) return fail(FLB_ERR_UNSUPPORTED, at + ": rows wider than " + std::to_string(widest) + " are not supported");
  if (G > 65535) return fail(FLB_ERR_UNSUPPORTED, at + ": more than 65535 groups are not supported");
  if (R > INT32_MAX || G * R > INT32_MAX) return fail(FLB_ERR_SHAPE, at + ": too many rows");
  const size_t ws = w || b ? (size_t)dtype_size(wdtype) : 1;
  if (off(w, ws) || off(b, ws)) return fail(FLB_ERR_ALIGN, at + ": weight and bias must be aligned to their element size");
  *empty = G * R == 0;
  return FLB_OK;
}

// A kept form: both arrays or neither, codes on 16 bytes.
int check_kept(const char* what, const int8_t* codes, const uint8_t* exps, bool needed) {
  const std::string at(what);
  if (!codes != !exps) return fail(FLB_ERR_SHAPE, at + ": codes and exps go together");
  if (needed && !codes) return fail(FLB_ERR_SHAPE, at + ": null codes");
  if (off(codes, 16)) return fail(FLB_ERR_ALIGN, at + ": codes must be 16-byte aligned");
  return FLB_OK;
}

int check_rows(const char* what, int64_t R, int64_t D, int dtype) {
  const std::string at(what);
  if (dtype_size(dtype) == 0) return fail(FLB_ERR_DTYPE, at + ": dtype must be f32, f16 or bf16");
  if (R < 0 || D < 1) return fail(FLB_ERR_SHAPE, at + ": R >= 0 and D >= 1 required");
  if (D > INT32_MAX / 2) return fail(FLB_ERR_UNSUPPORTED, at + ": rows this wide are not supported");
  if (R > INT64_MAX / 8 / (D + 256)) return fail(FLB_ERR_SHAPE, at + ": too many rows");
  return FLB_OK;
}

constexpr int64_t kWidestInt8 = 32768;  // a row's elements: 32768 * 127^2 < 2^31

// The sizes of an 8-bit product: within what the grid, the tensor maps and 32-bit sums hold.
int check_product(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 1) return fail(FLB_ERR_SHAPE, "int8_linear: M, N >= 0 and K >= 1 required");
  if (K > kWidestInt8) return fail(FLB_ERR_UNSUPPORTED, "int8_linear: rows wider than 32768 are not supported");
  if (M > INT32_MAX - 1024 || N > INT32_MAX - 1024 || (M > 0 && N > ((int64_t)1 << 44) / M))
    return fail(FLB_ERR_SHAPE, "int8_linear: too many rows");
  return FLB_OK;
}

int int8_linear_checked(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale, const int8_t* w_codes,
                        int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out, int64_t M, int64_t N,
                        int64_t K, int dtype, void* workspace, size_t workspace_bytes, int check_timeout, int drop, uint32_t limit,
                        void* stream) {
  if (dtype_size(dtype) == 0) return fail(FLB_ERR_DTYPE, "int8_linear: dtype must be f32, f16 or bf16");
  if (bias && bias_dtype != FLB_F32 && bias_dtype != dtype)
    return fail(FLB_ERR_DTYPE, "int8_linear: the bias must be float32 or of the output's dtype");
  int st = check_product(M, N, K);
  if (st != FLB_OK) return st;
  if (M == 0 || N == 0) return FLB_OK;
  if (!x == !x_codes || !x_codes != !x_scale) return fail(FLB_ERR_SHAPE, "int8_linear: either x, or x_codes and x_scale");
  if (!w_codes || !w_scale || !out) return fail(FLB_ERR_SHAPE, "int8_linear: null weight or out");
  if (x ? ldx < 0 : ldc < K) return fail(FLB_ERR_SHAPE, "int8_linear: bad row pitch of x");
  if (ldw < K) return fail(FLB_ERR_SHAPE, "int8_linear: bad row pitch of the weight");
  if (off(w_codes, 16) || ldw % 16 || (x_codes && (off(x_codes, 16) || ldc % 16)))
    return fail(FLB_ERR_ALIGN, "int8_linear: codes must start every row on 16 bytes");
  const size_t es = (size_t)dtype_size(dtype);
  if (off(x, es) || off(out, es) || off(w_scale, 4) || off(x_scale, 4) || off(bias, bias ? (size_t)dtype_size(bias_dtype) : 1))
    return fail(FLB_ERR_ALIGN, "int8_linear: pointers must be aligned to their element size");
  const size_t need = int8_linear_workspace_bytes(M, N, K, x != nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(FLB_ERR_WORKSPACE, "int8_linear: workspace smaller than flb_int8_linear_workspace_bytes()");
  if (off(workspace, 256)) return fail(FLB_ERR_ALIGN, "int8_linear: workspace must be 256-byte aligned");
  if (check_timeout) {
    cudaStreamCaptureStatus capture;
    if ((st = check_cuda(cudaStreamIsCapturing(as_stream(stream), &capture), "int8_linear capture status")) != FLB_OK) return st;
    if (capture != cudaStreamCaptureStatusNone)
      return fail(FLB_ERR_UNSUPPORTED, "int8_linear: check_timeout waits for the product, which a stream capture does not allow");
  }
  return int8_linear(x, ldx, x_codes, ldc, x_scale, w_codes, ldw, w_scale, bias, bias_dtype, out, M, N, K, dtype, workspace,
                     check_timeout, drop, limit, as_stream(stream));
}

}  // namespace
}  // namespace flb

using namespace flb;

extern "C" {

int64_t flb_code_pitch(int64_t D) { return D < 1 ? 0 : rows::code_pitch(D); }
int64_t flb_kept_blocks(int64_t D) { return D < 1 ? 0 : rows::blocks_of(D); }

int flb_layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, void* y, float* mean,
                       float* rstd, int8_t* codes, uint8_t* exps, int64_t G, int64_t R, int64_t D, int dtype,
                       float eps, void* stream) {
  bool empty;
  int st = check_norm("layer_norm_fwd", w, b, wdtype, G, R, D, ldx, dtype, 32768, &empty);
  if (st != FLB_OK) return st;
  if ((st = check_kept("layer_norm_fwd", codes, exps, false)) != FLB_OK) return st;
  if (empty) return FLB_OK;
  if (!x || !y) return fail(FLB_ERR_SHAPE, "layer_norm_fwd: null x or y");
  const size_t es = (size_t)dtype_size(dtype);
  if (off(x, es) || off(y, es) || off(mean, 4) || off(rstd, 4))
    return fail(FLB_ERR_ALIGN, "layer_norm_fwd: pointers must be aligned to their element size");
  return layer_norm_fwd(x, ldx, w, b, wdtype, y, mean, rstd, codes, exps, G, R, D, dtype, eps, as_stream(stream));
}

size_t flb_layer_norm_bwd_workspace_bytes(int64_t G, int64_t R, int64_t D) {
  if (G < 1 || R < 1 || D < 1 || D > 16384) return 0;
  return layer_norm_bwd_workspace_bytes(G, R, D);
}

int flb_layer_norm_bwd(const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps, const float* mean,
                       const float* rstd, const void* w, int wdtype, const void* dy, void* dx, void* dw, void* db,
                       int64_t G, int64_t R, int64_t D, int dtype, void* workspace, size_t workspace_bytes,
                       void* stream) {
  bool empty;
  int st = check_norm("layer_norm_bwd", w ? w : dw, w ? w : db, wdtype, G, R, D, ldx, dtype, 16384, &empty);
  if (st != FLB_OK) return st;
  if ((st = check_kept("layer_norm_bwd", codes, exps, false)) != FLB_OK) return st;
  if (!dw != !db) return fail(FLB_ERR_SHAPE, "layer_norm_bwd: dw and db go together");
  const size_t ws = dw ? (size_t)dtype_size(wdtype) : 1;
  if (off(dw, ws) || off(db, ws)) return fail(FLB_ERR_ALIGN, "layer_norm_bwd: dw and db must be aligned to their element size");
  cudaStream_t s = as_stream(stream);
  if (empty) {  // sums over no rows
    if (dw && G > 0) {
      if ((st = check_cuda(cudaMemsetAsync(dw, 0, G * D * ws, s), "layer_norm_bwd dw reset")) != FLB_OK) return st;
      return check_cuda(cudaMemsetAsync(db, 0, G * D * ws, s), "layer_norm_bwd db reset");
    }
    return FLB_OK;
  }
  if (!dy || !dx || !rstd || (!codes && (!x || !mean))) return fail(FLB_ERR_SHAPE, "layer_norm_bwd: null input or output");
  const size_t es = (size_t)dtype_size(dtype);
  if (off(x, es) || off(dy, es) || off(dx, es) || off(mean, 4) || off(rstd, 4))
    return fail(FLB_ERR_ALIGN, "layer_norm_bwd: pointers must be aligned to their element size");
  const size_t need = dw ? layer_norm_bwd_workspace_bytes(G, R, D) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(FLB_ERR_WORKSPACE, "layer_norm_bwd: workspace smaller than flb_layer_norm_bwd_workspace_bytes()");
  if (off(workspace, 16)) return fail(FLB_ERR_ALIGN, "layer_norm_bwd: workspace must be 16-byte aligned");
  return layer_norm_bwd(x, ldx, codes, exps, mean, rstd, w, wdtype, dy, dx, dw, db, G, R, D, dtype, workspace, s);
}

int flb_layer_norm_int8(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, int8_t* codes, float* scale,
                        int64_t G, int64_t R, int64_t D, int dtype, float eps, void* stream) {
  bool empty;
  int st = check_norm("layer_norm_int8", w, b, wdtype, G, R, D, ldx, dtype, kWidestInt8, &empty);
  if (st != FLB_OK || empty) return st;
  if (!x || !codes || !scale) return fail(FLB_ERR_SHAPE, "layer_norm_int8: null x, codes or scale");
  if (off(x, (size_t)dtype_size(dtype)) || off(codes, 16) || off(scale, 4))
    return fail(FLB_ERR_ALIGN, "layer_norm_int8: codes must be 16-byte aligned, x and scale to their element size");
  return layer_norm_int8(x, ldx, w, b, wdtype, codes, scale, G, R, D, dtype, eps, as_stream(stream));
}

int flb_int8_rows(const void* x, int64_t ldx, int8_t* codes, float* scale, int64_t R, int64_t D, int dtype, void* stream) {
  bool empty;
  int st = check_norm("int8_rows", nullptr, nullptr, dtype, 1, R, D, ldx, dtype, kWidestInt8, &empty);
  if (st != FLB_OK || empty) return st;
  if (!x || !codes || !scale) return fail(FLB_ERR_SHAPE, "int8_rows: null x, codes or scale");
  if (off(x, (size_t)dtype_size(dtype)) || off(codes, 16) || off(scale, 4))
    return fail(FLB_ERR_ALIGN, "int8_rows: codes must be 16-byte aligned, x and scale to their element size");
  return int8_rows(x, ldx, codes, scale, R, D, dtype, nullptr, 0, as_stream(stream));
}

size_t flb_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_is_codes) {
  if (check_product(M, N, K) != FLB_OK || M == 0 || N == 0) return 0;
  return int8_linear_workspace_bytes(M, N, K, !x_is_codes);
}

int flb_int8_linear(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale,
                    const int8_t* w_codes, int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out,
                    int64_t M, int64_t N, int64_t K, int dtype, void* workspace, size_t workspace_bytes, int check_timeout,
                    void* stream) {
  return int8_linear_checked(x, ldx, x_codes, ldc, x_scale, w_codes, ldw, w_scale, bias, bias_dtype, out, M, N, K, dtype, workspace,
                             workspace_bytes, check_timeout, -1, 0, stream);
}

int flb_int8_linear_wait_test(const void* x, int64_t ldx, const int8_t* x_codes, int64_t ldc, const float* x_scale,
                              const int8_t* w_codes, int64_t ldw, const float* w_scale, const void* bias, int bias_dtype, void* out,
                              int64_t M, int64_t N, int64_t K, int dtype, void* workspace, size_t workspace_bytes, int check_timeout,
                              int64_t drop_step, uint32_t spin_limit, void* stream) {
  if (drop_step < -1 || drop_step > INT32_MAX || spin_limit < 1)
    return fail(FLB_ERR_SHAPE, "int8_linear wait test: drop_step >= -1 and spin_limit >= 1 required");
  return int8_linear_checked(x, ldx, x_codes, ldc, x_scale, w_codes, ldw, w_scale, bias, bias_dtype, out, M, N, K, dtype, workspace,
                             workspace_bytes, check_timeout, (int)drop_step, spin_limit, stream);
}

int flb_pack8(const void* x, int8_t* codes, uint8_t* exps, int64_t R, int64_t D, int dtype, void* stream) {
  int st = check_rows("pack8", R, D, dtype);
  if (st != FLB_OK) return st;
  if ((st = check_kept("pack8", codes, exps, R > 0)) != FLB_OK) return st;
  if (R == 0) return FLB_OK;
  if (!x) return fail(FLB_ERR_SHAPE, "pack8: null x");
  if (off(x, (size_t)dtype_size(dtype))) return fail(FLB_ERR_ALIGN, "pack8: x must be aligned to its element size");
  return pack8(x, codes, exps, R, D, dtype, as_stream(stream));
}

int flb_unpack8(const int8_t* codes, const uint8_t* exps, void* out, int64_t R, int64_t D, int dtype, void* stream) {
  int st = check_rows("unpack8", R, D, dtype);
  if (st != FLB_OK) return st;
  if ((st = check_kept("unpack8", codes, exps, R > 0)) != FLB_OK) return st;
  if (R == 0) return FLB_OK;
  if (!out) return fail(FLB_ERR_SHAPE, "unpack8: null out");
  if (off(out, (size_t)dtype_size(dtype))) return fail(FLB_ERR_ALIGN, "unpack8: out must be aligned to its element size");
  return unpack8(codes, exps, out, R, D, dtype, as_stream(stream));
}

int flb_gate_fwd(const void* x, const void* z, void* y, int8_t* cx, uint8_t* ex, int8_t* cz, uint8_t* ez, int64_t R,
                 int64_t D, int dtype, void* stream) {
  int st = check_rows("gate_fwd", R, D, dtype);
  if (st != FLB_OK) return st;
  if ((st = check_kept("gate_fwd", cx, ex, false)) != FLB_OK || (st = check_kept("gate_fwd", cz, ez, false)) != FLB_OK)
    return st;
  if (!cx != !cz) return fail(FLB_ERR_SHAPE, "gate_fwd: x and z are kept together");
  if (R == 0) return FLB_OK;
  if (!x || !z || !y) return fail(FLB_ERR_SHAPE, "gate_fwd: null x, z or y");
  const size_t es = (size_t)dtype_size(dtype);
  if (off(x, es) || off(z, es) || off(y, es)) return fail(FLB_ERR_ALIGN, "gate_fwd: pointers must be aligned to their element size");
  return gate_fwd(x, z, y, cx, ex, cz, ez, R, D, dtype, as_stream(stream));
}

int flb_gate_bwd(const void* x, const void* z, const int8_t* cx, const uint8_t* ex, const int8_t* cz,
                 const uint8_t* ez, const void* dy, void* dx, void* dz, int64_t R, int64_t D, int dtype, void* stream) {
  int st = check_rows("gate_bwd", R, D, dtype);
  if (st != FLB_OK) return st;
  if ((st = check_kept("gate_bwd", cx, ex, false)) != FLB_OK || (st = check_kept("gate_bwd", cz, ez, false)) != FLB_OK)
    return st;
  if (!cx != !cz) return fail(FLB_ERR_SHAPE, "gate_bwd: x and z are kept together");
  if (R == 0) return FLB_OK;
  if (!dy || !dx || !dz || (!cx && (!x || !z))) return fail(FLB_ERR_SHAPE, "gate_bwd: null input or output");
  const size_t es = (size_t)dtype_size(dtype);
  if (off(x, es) || off(z, es) || off(dy, es) || off(dx, es) || off(dz, es))
    return fail(FLB_ERR_ALIGN, "gate_bwd: pointers must be aligned to their element size");
  return gate_bwd(x, z, cx, ex, cz, ez, dy, dx, dz, R, D, dtype, as_stream(stream));
}

}  // extern "C"
