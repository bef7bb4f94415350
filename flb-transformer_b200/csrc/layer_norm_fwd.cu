// Row kernels that read a row once and write one: LayerNorm forward (with its rows kept in 8 bits on
// request), LayerNorm to 8-bit integer rows, and plain rows to 8-bit integer rows.
//
//   mean = sum(x) / D,  var = sum((x - mean)^2) / D,  h = (x - mean) / sqrt(var + eps),  y = h w + b
//   integer rows of v: a = max |v|, code = round(v * (127 / a)), scale = a / 127
//
// Bound by memory: a row is read and written once. It stays in registers between its statistics and its
// output, so the variance is the second moment about the mean itself, not a difference of large sums. A
// warp takes a row of up to 1024 elements and needs no barrier; wider rows get a block each, 32 elements a
// thread. The weight and bias are re-read for every row: they stay in L1.
#include "rows.cuh"

namespace flb {

using namespace rows;

namespace {

enum { OUT_Y = 0, OUT_KEPT = 1, OUT_INT8 = 2 };

struct RowArgs {
  const void* x;
  int64_t ldx;  // elements
  const void *w, *b;
  bool w32;  // w and b are float32 (else x's type)
  void* y;
  float *mean, *rstd;  // null: not wanted
  int8_t* codes;       // OUT_KEPT: h; OUT_INT8: the row
  uint8_t* exps;
  float* scale;
  int64_t rows, rows_per_group;
  int D;
  float eps;
  uint32_t* zero;  // words that a kernel after this one counts in
  int64_t n_zero;
};

// `fill` where there is no such vector
template <typename T, bool VEC>
__device__ __forceinline__ void load_param(F2 (&v)[4], const void* p, bool f32, float fill, int64_t off, int base,
                                           int lane, int D) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f2(fill);
  } else if (f32) {
    load8<float, VEC>(v, reinterpret_cast<const float*>(p) + off, base, lane, D);
  } else {
    load8<T, VEC>(v, reinterpret_cast<const T*>(p) + off, base, lane, D);
  }
}

// Zeros in the place of a chunk's elements at or beyond D
template <bool VEC> __device__ __forceinline__ void zero_beyond(F2 (&v)[4], int base, int lane, int D) {
  if (Chunk<VEC>::has(base, lane, 7, D)) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 r = split(v[i]);
    v[i] = f2(Chunk<VEC>::has(base, lane, 2 * i, D) ? r.x : 0.f, Chunk<VEC>::has(base, lane, 2 * i + 1, D) ? r.y : 0.f);
  }
}

template <typename T, bool VEC, bool WARP, int CH, bool NORM, int OUT>
__global__ void __launch_bounds__(WARP ? 256 : 1024) row_fwd_kernel(const RowArgs a) {
  __shared__ float slot[WARP ? 1 : 3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (!NORM) {
    let_successor_start();
    if (blockIdx.x == 0)
      for (int64_t i = threadIdx.x; i < a.n_zero; i += blockDim.x) a.zero[i] = 0;
  }
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  if (row >= a.rows) return;
  const int D = a.D;
  // chunk c of this warp starts at first + c * step
  const int first = WARP ? 0 : warp * 256, step = WARP ? 256 : (int)blockDim.x * 8;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  Raw8<T> raw[CH];  // as loaded: fewer registers for 16-bit rows, so more rows in flight
#pragma unroll
  for (int c = 0; c < CH; ++c) load_raw<T, VEC>(raw[c], x, first + c * step, lane, D);
  float mean = 0.f, rstd = 1.f;
  if constexpr (NORM) {
    F2 s = f2(0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 v[4];
      to_float<T>(raw[c], v);
      s = add2(s, add2(add2(v[0], v[1]), add2(v[2], v[3])));
    }
    mean = row_sum<WARP>(sum2(s), slot[0]) / D;
    s = f2(0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      F2 v[4];
      to_float<T>(raw[c], v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = add2(v[i], f2(-mean));
      zero_beyond<VEC>(v, first + c * step, lane, D);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fma2(v[i], v[i], s);
    }
    rstd = 1.f / sqrtf(row_sum<WARP>(sum2(s), slot[WARP ? 0 : 1]) / D + a.eps);
    if (threadIdx.x == 0 || (WARP && lane == 0)) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
  const int64_t param = NORM && a.rows_per_group != a.rows ? row / a.rows_per_group * D : 0;
  // the normalised chunk, then with the weight and bias (beyond the row: anything)
  auto normalised = [&](int c, F2 (&v)[4]) {
    to_float<T>(raw[c], v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(add2(v[i], f2(-mean)), f2(rstd));
  };
  auto affine = [&](int c, F2 (&v)[4]) {
    F2 w[4], b[4];
    load_param<T, VEC>(w, a.w, a.w32, 1.f, param, first + c * step, lane, D);
    load_param<T, VEC>(b, a.b, a.w32, 0.f, param, first + c * step, lane, D);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fma2(v[i], w[i], b[i]);
  };
  if constexpr (OUT != OUT_INT8) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int base = first + c * step;
      F2 v[4];
      normalised(c, v);
      if constexpr (OUT == OUT_KEPT) {
        if (base < D) {
          zero_beyond<VEC>(v, base, lane, D);
          // a row with an infinity or NaN has NaN throughout, so a block's values are all NaN or none
          uint32_t m[VEC ? 1 : 2];
          max_bits<VEC>(v, m);
          keep8<VEC>(v, m, a.codes + row * code_pitch(D), a.exps + row * blocks_of(D), base, lane, D);
        }
      }
      affine(c, v);
      store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * D, v, base, lane, D);
    }
  } else {
    uint32_t m = 0;
    F2 v[NORM ? CH : 1][4];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (NORM) {
        normalised(c, v[c]);
        affine(c, v[c]);
        zero_beyond<VEC>(v[c], first + c * step, lane, D);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r = split(v[c][i]);
          m = __vimax3_u32(m, abs_bits(r.x), abs_bits(r.y));
        }
      } else {
        uint32_t h[1];
        max_bits<T, true>(raw[c], h);
        m = max(m, h[0]);
      }
    }
    m = row_max<WARP>(m, reinterpret_cast<uint32_t*>(slot[WARP ? 0 : 2]));
    // An infinity or NaN in the row makes its scale, and so all that is computed with it, NaN. Below
    // 2^-118 the factor 127 / a would be infinite: such a row counts as zeros.
    const float amax = __uint_as_float(m);
    const bool bad = m >= 0x7f800000u;
    const float f = bad || amax < 3.0092655e-36f ? 0.f : 127.f / amax;
    if (threadIdx.x == 0 || (WARP && lane == 0)) a.scale[row] = bad ? __uint_as_float(0x7fffffffu) : amax / 127.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint32_t q[8];
      F2 u[4];
      if constexpr (!NORM) to_float<T>(raw[c], u);
      float t[8];
      to_scalars(NORM ? v[NORM ? c : 0] : u, t);
      // product and rounding apart, each rounded as written above (as a packed pair they come out as one
      // multiply-add, with another code now and then)
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = f == 0.f ? 0u : code_of(__fmul_rn(t[j], f));
      store_codes<VEC>(a.codes + row * code_pitch(D), q, first + c * step, lane, D);
    }
  }
}

template <typename T, bool VEC, bool NORM, int OUT>
int launch_rows(const RowArgs& a, cudaStream_t s) {
  const int D = a.D;
  if (D <= 1024) {
    // few rows: a warp a block, so that they spread over the SMs; many: eight, fewer blocks to start
    const int warps = a.rows >= 16 * (int64_t)num_sms() ? 8 : a.rows >= 4 * (int64_t)num_sms() ? 4 : 1;
    const dim3 grid((unsigned)((a.rows + warps - 1) / warps)), block(32 * warps);
    switch ((D + 255) / 256) {
      case 1: row_fwd_kernel<T, VEC, true, 1, NORM, OUT><<<grid, block, 0, s>>>(a); break;
      case 2: row_fwd_kernel<T, VEC, true, 2, NORM, OUT><<<grid, block, 0, s>>>(a); break;
      case 3: row_fwd_kernel<T, VEC, true, 3, NORM, OUT><<<grid, block, 0, s>>>(a); break;
      default: row_fwd_kernel<T, VEC, true, 4, NORM, OUT><<<grid, block, 0, s>>>(a); break;
    }
  } else {
    row_fwd_kernel<T, VEC, false, 4, NORM, OUT><<<(unsigned)a.rows, 32 * ((D + 1023) / 1024), 0, s>>>(a);
  }
  count_launches(1);
  return check_cuda(cudaGetLastError(), "row kernel launch");
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <bool NORM, int OUT> int dispatch_rows(const RowArgs& a, int dtype, cudaStream_t s) {
  const int es = dtype_size(dtype);
  const bool vec = a.D % 8 == 0 && a.ldx * es % 16 == 0 && on16(a.x) && on16(a.y) && on16(a.w) && on16(a.b) && on16(a.codes);
  switch (dtype) {
    case FLB_F32: return vec ? launch_rows<float, true, NORM, OUT>(a, s) : launch_rows<float, false, NORM, OUT>(a, s);
    case FLB_F16: return vec ? launch_rows<__half, true, NORM, OUT>(a, s) : launch_rows<__half, false, NORM, OUT>(a, s);
    default: return vec ? launch_rows<__nv_bfloat16, true, NORM, OUT>(a, s) : launch_rows<__nv_bfloat16, false, NORM, OUT>(a, s);
  }
}

}  // namespace

int layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, void* y, float* mean,
                   float* rstd, int8_t* codes, uint8_t* exps, int64_t G, int64_t R, int64_t D, int dtype, float eps,
                   cudaStream_t s) {
  const RowArgs a{x, ldx, w, b, wdtype == FLB_F32, y, mean, rstd, codes, exps, nullptr, G * R, R, (int)D, eps, nullptr, 0};
  return codes ? dispatch_rows<true, OUT_KEPT>(a, dtype, s) : dispatch_rows<true, OUT_Y>(a, dtype, s);
}

int layer_norm_int8(const void* x, int64_t ldx, const void* w, const void* b, int wdtype, int8_t* codes, float* scale,
                    int64_t G, int64_t R, int64_t D, int dtype, float eps, cudaStream_t s) {
  const RowArgs a{x, ldx, w, b, wdtype == FLB_F32, nullptr, nullptr, nullptr, codes, nullptr, scale, G * R, R, (int)D, eps, nullptr, 0};
  return dispatch_rows<true, OUT_INT8>(a, dtype, s);
}

int int8_rows(const void* x, int64_t ldx, int8_t* codes, float* scale, int64_t R, int64_t D, int dtype, uint32_t* zero,
              int64_t n_zero, cudaStream_t s) {
  const RowArgs a{x, ldx, nullptr, nullptr, false, nullptr, nullptr, nullptr, codes, nullptr, scale, R, R, (int)D, 0.f, zero, n_zero};
  return dispatch_rows<false, OUT_INT8>(a, dtype, s);
}

}  // namespace flb
