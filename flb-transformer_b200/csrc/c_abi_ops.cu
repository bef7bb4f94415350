// extern "C" boundary of the row operators: LayerNorm, the 8-bit kept form, the sigmoid gate.
#include "common.cuh"
#include "rows.cuh"

namespace flb {

int layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, void* y, float* mean,
                   float* rstd, int8_t* codes, uint8_t* exps, int64_t G, int64_t R, int64_t D, int dtype, float eps,
                   cudaStream_t s);
size_t layer_norm_bwd_workspace_bytes(int64_t G, int64_t R, int64_t D, int dtype);
int layer_norm_bwd(const void* x, int64_t ldx, const int8_t* codes, const uint8_t* exps, const float* mean,
                   const float* rstd, const void* w, int wdtype, const void* dy, void* dx, void* dw, void* db, int64_t G,
                   int64_t R, int64_t D, int dtype, void* ws, cudaStream_t s);
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

size_t flb_layer_norm_bwd_workspace_bytes(int64_t G, int64_t R, int64_t D, int dtype) {
  if (G < 1 || R < 1 || D < 1 || D > 16384) return 0;
  return layer_norm_bwd_workspace_bytes(G, R, D, dtype);
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
  const size_t need = dw ? layer_norm_bwd_workspace_bytes(G, R, D, dtype) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(FLB_ERR_WORKSPACE, "layer_norm_bwd: workspace smaller than flb_layer_norm_bwd_workspace_bytes()");
  if (off(workspace, 16)) return fail(FLB_ERR_ALIGN, "layer_norm_bwd: workspace must be 16-byte aligned");
  return layer_norm_bwd(x, ldx, codes, exps, mean, rstd, w, wdtype, dy, dx, dw, db, G, R, D, dtype, workspace, s);
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
