// Row kernels that read a row once and write one: LayerNorm forward (with its rows kept in 8 bits on
// request), LayerNorm to 8-bit integer rows, and plain rows to 8-bit integer rows.
//
//   mean = sum(x) / D,  var = sum((x - mean)^2) / D,  h = (x - mean) / sqrt(var + eps),  y = h w + b
//   integer rows of v: a = max |v|, code = round(v * (127 / a)), scale = a / 127
//
// Bound by memory: a row is read and written once. It stays in registers between its statistics and its
// output, so the variance is the second moment about the mean itself, not a difference of large sums. A
// warp takes a row of up to 1024 elements and needs no barrier; a wider one gets a block, 16 elements a
// thread (32 beyond 8192). A block walks over rows a fixed distance apart, the next rows on their way to shared
// memory meanwhile, the weight and bias there as float32 (in registers they cost a third of the warps: 129 us
// against 105 for 32768 x 4096 bfloat16, which is 5.1 TB/s of reads and writes; re-read and converted for each
// row 136).
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
template <typename T, Layout L>
__device__ __forceinline__ void load_param(F2 (&v)[4], const void* p, bool f32, float fill, int64_t off, int base,
                                           int lane, int D) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f2(fill);
  } else if (f32) {
    load8<float, L>(v, reinterpret_cast<const float*>(p) + off, base, lane, D);
  } else {
    load8<T, L>(v, reinterpret_cast<const T*>(p) + off, base, lane, D);
  }
}

// Rows held at a time, the present one included: with the widest rows one
template <int CH, int MODE> constexpr int kStages = MODE == 2 ? 1 : 2;
constexpr int kWarps = 4;  // of a block whose warps have a row each
template <int MODE> constexpr int kMostThreads = MODE == 0 ? 32 * kWarps : MODE == 1 ? 512 : 1024;

// MODE 0: a warp a row (D <= 1024), 1: a block a row (D <= 8192), 2: a block of up to 1024 threads
template <typename T, bool VEC, int MODE, int CH, bool NORM, int OUT>
__global__ void __launch_bounds__(kMostThreads<MODE>, 1024 / kMostThreads<MODE>) row_fwd_kernel(const RowArgs a) {
  constexpr Layout L = kLayout<T, VEC>;
  constexpr bool WARP = MODE == 0;
  constexpr bool PARAMS = NORM && MODE != 2;  // the weight and bias stay in shared memory, as float32
  constexpr int S = kStages<CH, MODE>;
  // [CH][4][threads, or lanes of a warp's row] float4: weight and bias | [S][CH] chunks of rows
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float slot[WARP ? 1 : 2][3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (OUT == OUT_INT8) let_successor_start();  // the product that reads the rows
  if constexpr (!NORM) {
    if (blockIdx.x == 0)
      for (int64_t i = threadIdx.x; i < a.n_zero; i += blockDim.x) a.zero[i] = 0;
  }
  const int D = a.D;
  // chunk c of this warp starts at first + c * 256
  const int first = WARP ? 0 : warp * 256 * CH;
  const int64_t stride = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  const int64_t row0 = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  const int64_t group = blockIdx.y, rows = a.rows_per_group;
  const T* const x = reinterpret_cast<const T*>(a.x) + group * rows * a.ldx;
  const int param_threads = WARP ? 32 : (int)blockDim.x, param_thread = WARP ? lane : (int)threadIdx.x;
  float4* const params = reinterpret_cast<float4*>(dyn) + param_thread;
  uint8_t* const ring = dyn + (PARAMS ? (size_t)CH * 64 * param_threads : 0);
  auto chunk_at = [&](int stage, int c) { return ring + (size_t)(stage * CH + c) * copy_bytes<T, L>(blockDim.x); };
  auto issue = [&](int64_t r, int stage) {
    if (r < rows) {
#pragma unroll
      for (int c = 0; c < CH; ++c) copy8<T, L>(chunk_at(stage, c), x + r * a.ldx, first + c * 256, lane, D);
    }
    copies_commit();
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) issue(row0 + k * stride, k);
  if constexpr (!WARP) {
    if (warp == 0)
      for (int i = 0; i < 6; ++i) slot[i / 3][i % 3][lane] = 0.f;
  }
  if constexpr (PARAMS) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (WARP && c % (int)(blockDim.x >> 5) != warp) continue;
      F2 w[4], b[4];
      load_param<T, L>(w, a.w, a.w32, 1.f, group * D, first + c * 256, lane, D);
      load_param<T, L>(b, a.b, a.w32, 0.f, group * D, first + c * 256, lane, D);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 lo = split(k < 2 ? w[2 * k] : b[2 * k - 4]), hi = split(k < 2 ? w[2 * k + 1] : b[2 * k - 3]);
        params[(c * 4 + k) * param_threads] = make_float4(lo.x, lo.y, hi.x, hi.y);
      }
    }
  }
  __syncthreads();

  int stage = 0, turn = 0;
  for (int64_t r = row0; r < rows; r += stride) {
    meet_copies<L>();
    issue(r + (S - 1) * stride, stage == 0 ? S - 1 : stage - 1);  // where the row before this one was
    const int64_t row = group * rows + r;
    // the chunks' elements, and as they were loaded (for the largest magnitudes of plain rows)
    F2 v[CH][4];
    Raw8<T> raw[NORM ? 1 : CH];
    copies_wait<S - 1>();
    meet_copies<L>();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      Raw8<T>& u = raw[NORM ? 0 : c];
      copied_raw<T, L>(chunk_at(stage, c), u, x + r * a.ldx, first + c * 256, lane, D);
      to_float<T>(u, v[c]);
    }
    if constexpr (NORM) {
      F2 s = f2(0.f);
#pragma unroll
      for (int c = 0; c < CH; ++c) s = add2(s, add2(add2(v[c][0], v[c][1]), add2(v[c][2], v[c][3])));
      const float mean = row_sum<WARP>(sum2(s), slot[turn][0]) / D;
      s = f2(0.f);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = add2(v[c][i], f2(-mean));
        zero_beyond<L>(v[c], first + c * 256, lane, D);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fma2(v[c][i], v[c][i], s);
      }
      const float rstd = 1.f / sqrtf(row_sum<WARP>(sum2(s), slot[turn][WARP ? 0 : 1]) / D + a.eps);
      if (threadIdx.x == 0 || (WARP && lane == 0)) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int base = first + c * 256;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = mul2(v[c][i], f2(rstd));
        if constexpr (OUT == OUT_KEPT) {
          if (base < D) {
            // a row with an infinity or NaN, or whose sum is one, has NaN throughout
            uint32_t m[L == EIGHT ? 1 : 2];
            max_bits<L>(v[c], m);
            keep8<L>(v[c], m, a.codes + row * code_pitch(D), a.exps + row * blocks_of(D), base, lane, D);
          }
        }
        F2 w[4], b[4];
        if constexpr (PARAMS) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float4 u = params[(c * 4 + k) * param_threads], t = params[(c * 4 + 2 + k) * param_threads];
            w[2 * k] = f2(u.x, u.y), w[2 * k + 1] = f2(u.z, u.w);
            b[2 * k] = f2(t.x, t.y), b[2 * k + 1] = f2(t.z, t.w);
          }
        } else {
          load_param<T, L>(w, a.w, a.w32, 1.f, group * D, base, lane, D);
          load_param<T, L>(b, a.b, a.w32, 0.f, group * D, base, lane, D);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = fma2(v[c][i], w[i], b[i]);
        if constexpr (OUT != OUT_INT8) store8<T, L>(reinterpret_cast<T*>(a.y) + row * D, v[c], base, lane, D);
      }
    }
    if constexpr (OUT == OUT_INT8) {
      uint32_t m = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if constexpr (NORM) {
          zero_beyond<L>(v[c], first + c * 256, lane, D);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 r = split(v[c][i]);
            m = __vimax3_u32(m, abs_bits(r.x), abs_bits(r.y));
          }
        } else {
          uint32_t h[1];
          max_bits<T, EIGHT>(raw[c], h);
          m = max(m, h[0]);
        }
      }
      m = row_max<WARP>(m, reinterpret_cast<uint32_t*>(slot[turn][WARP ? 0 : 2]));
      const float factor = int8_factor(m);
      if (threadIdx.x == 0 || (WARP && lane == 0)) a.scale[row] = int8_scale(m);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t q[8];
        int8_codes(v[c], factor, q);
        store_codes<L>(a.codes + row * code_pitch(D), q, first + c * 256, lane, D);
      }
    }
    // a warp that is a row ahead writes the other slots, and is not two ahead before every warp has passed
    // a barrier of the row between, after reading this one's
    if constexpr (!WARP) turn ^= 1;
    if constexpr (S > 1) stage = stage + 1 == S ? 0 : stage + 1;
  }
}

template <typename T, bool VEC, int MODE, int CH, bool NORM, int OUT> int launch_mode(const RowArgs& a, int threads, cudaStream_t s) {
  auto k = row_fwd_kernel<T, VEC, MODE, CH, NORM, OUT>;
  const size_t ring = (size_t)kStages<CH, MODE> * CH * copy_bytes<T, kLayout<T, VEC>>(threads);
  const size_t smem = ring + (NORM && MODE != 2 ? (size_t)CH * 64 * (MODE == 0 ? 32 : threads) : 0);
  const int st = ensure_dyn_smem(reinterpret_cast<const void*>(k), (int)smem, "row kernel shared memory");
  if (st != FLB_OK) return st;
  // as many blocks as an SM holds (64 registers a thread, 224 KB), each with as many rows as the others
  const int64_t at_once = MODE == 0 ? threads / 32 : 1, groups = a.rows / a.rows_per_group;
  const int64_t units = (a.rows_per_group + at_once - 1) / at_once;
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(1024 / threads, (224 << 10) / (int64_t)(smem + 2048)));
  const int64_t room = std::max<int64_t>(1, num_sms() * per_sm / groups);
  k<<<dim3((unsigned)std::min(units, room), (unsigned)groups), threads, smem, s>>>(a);
  count_launches(1);
  return check_cuda(cudaGetLastError(), "row kernel launch");
}

template <typename T, bool VEC, bool NORM, int OUT> int launch_rows(const RowArgs& a, cudaStream_t s) {
  const int D = a.D;
  if (D <= 1024) {
    // few rows: a warp a block, so that they spread over the SMs
    const int threads = a.rows >= 4 * (int64_t)num_sms() ? 32 * kWarps : 32;
    switch ((D + 255) / 256) {
      case 1: return launch_mode<T, VEC, 0, 1, NORM, OUT>(a, threads, s);
      case 2: return launch_mode<T, VEC, 0, 2, NORM, OUT>(a, threads, s);
      case 3: return launch_mode<T, VEC, 0, 3, NORM, OUT>(a, threads, s);
      default: return launch_mode<T, VEC, 0, 4, NORM, OUT>(a, threads, s);
    }
  }
  if (D <= 8192) return launch_mode<T, VEC, 1, 2, NORM, OUT>(a, 32 * ((D + 511) / 512), s);
  return launch_mode<T, VEC, 2, 4, NORM, OUT>(a, 32 * ((D + 1023) / 1024), s);
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
